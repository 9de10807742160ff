// Sampling from given random numbers (btf_sample): temperature, top-k, top-p and
// min-p on one row of logits per thread-block cluster, whose shared memory holds the
// row: the logits are read once.
//
// All three filters keep a prefix of the order (logit descending, index
// ascending), so nothing is sorted: a cut (key, index) in that order plus a bound on
// the exponent is the kept set. What bounds the kernel is the number of passes over
// the row and of cluster barriers (about 0.7 us each), so the common cases take few:
//   top-k: a histogram of each thread's largest logit (of its 32 or so) gives a bound
//     that at least k logits reach and few more than k exceed; those go to the
//     cluster's first CTA, which ranks them exactly and finishes the row: 3 barriers;
//   top-p: a histogram of masses over 2048 bins of (max - l) / T gives the cut's bin.
//     Few elements down to it: the same finish. Else the bin's own elements are ranked
//     (or, when there are many, split further by the bits of their keys), and the
//     token comes from a walk over running masses in index order, each CTA over its
//     own part of the row;
//   no such filter: the walk alone: 2 barriers.
// Bounds on (max - l) / T are turned into bounds on keys once, so that a pass over the
// row compares integers and only what it keeps is worked out.
//
// Masses are 64-bit integers, w = rint(exp((l - max) / T) 2^S): sums are exact in
// any order, so the CTAs of a cluster, the histogram and the final walk agree on
// every total to the last bit, and the drawn token is a function of the inputs
// alone. S = 62 - ceil(log2 V) (44 for V up to 2^18): a mass is off by 2^-45 of
// the largest one; exponents are taken in 64 bits, since a token next to a border
// of the running mass would go the other way under the 2^-24 of fp32.
#include <algorithm>
#include <cmath>

#include "elem.cuh"
#include "sample.h"

namespace btf {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 2048;
constexpr int kCand = 512;     // elements that one CTA ranks exactly, one per thread
constexpr int kMaxCluster = 16;
constexpr float kSpan = 32.0f;  // exponents below -kSpan have mass 0: e^-32 < 2^-46

struct SampleParams {
  const void* x;
  int64_t ld;
  int type, V, chunk, S;  // chunk: logits per CTA, a multiple of 4 x kThreads
  const float *u, *temp, *top_p, *min_p;
  const int32_t* top_k;
  int32_t *tok, *tok2;
  float* logprob;
};

// Order-preserving key of a logit: larger key, larger logit; -0 as +0, NaN as -inf.
// Key 0 is no logit (what pads a chunk).
constexpr uint32_t kNegInf = 0x007fffffu;
__device__ __forceinline__ uint32_t key_of(float v) {
  if (v != v) return kNegInf;
  const uint32_t b = __float_as_uint(v + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// ---- distributed shared memory of the cluster
__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint64_t ld_cluster_u64(uint32_t a) {
  uint64_t v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void st_cluster_u64(uint32_t a, uint64_t v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(a), "l"(v) : "memory");
}
__device__ __forceinline__ uint32_t atom_cluster_inc(uint32_t a) {
  uint32_t v;
  asm volatile("atom.shared::cluster.add.u32 %0, [%1], 1;" : "=r"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_barrier() {
  __syncwarp();
  cluster_arrive_release();
  cluster_wait_acquire();
}

struct Shared {
  uint64_t slot[2][kMaxCluster][2];  // values that the CTAs send one another, in turn
  uint64_t group[kMaxCluster][kBins / 32];  // every CTA's sums of 32 bins
  uint64_t warp[kWarps][2];
  uint64_t found[2];
  int found_bin;
  double exp2_64[64];  // 2^(i / 64)
  uint64_t cmass[kCand];
  uint32_t ckey[kCand], cidx[kCand];
  uint32_t ncand;
};
// A histogram of counts or of masses. Its groups of 32 bins are summed for the whole cluster's use.
struct Hist {
  unsigned long long bin[kBins];
};

// One row's state, the same in every thread of the cluster.
struct Row {
  uint32_t top;     // key of the largest logit
  float top_value;
  double m, inv_t;  // the largest logit and 1 / T
  float bin_scale;
  double min_e;     // min-p: exponents below are dropped
  uint32_t alive;   // keys below have no mass
  int S;
  uint32_t cut_key, cut_idx;  // kept: key > cut_key, or == and idx <= cut_idx
  const double* table;

  __device__ __forceinline__ double exponent(uint32_t key) const {
    return key == top ? 0.0 : ((double)key_value(key) - m) * inv_t;
  }
  // (max - l) / T in bins: fp32 subtraction and product are monotone, so it follows the order. At least kBins, or
  // NaN, has no mass.
  __device__ __forceinline__ float place(uint32_t key) const {
    return key == top ? 0.0f : (top_value - key_value(key)) * bin_scale;
  }
  // rint(2^S e^x) for -33 < x <= 0 by a table of 2^(i / 64) and the Taylor polynomial of the rest (Tang's method):
  // x = n ln2 / 64 + r, |r| <= ln2 / 128, e^r to r^5 / 120 (the rest below 2^-54), in all within 2^-48 relative.
  __device__ __forceinline__ uint64_t weight_of(double x) const {
    constexpr double kRound = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to an integer
    const double big = fma(x, 92.332482616893656877, kRound);  // 64 / ln 2
    const int n = __double2loint(big);
    const double r = fma(big - kRound, -0.010830424696249145, x);  // ln 2 / 64
    double p = fma(r, 1.0 / 120, 1.0 / 24);
    p = fma(p, r, 1.0 / 6);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    const double t = table[n & 63];
    const double scaled = __hiloint2double(__double2hiint(t) + (((n >> 6) + S) << 20), __double2loint(t));
    // w <= 2^44: the low bits of w + 1.5 * 2^52 are w rounded
    return (uint64_t)__double_as_longlong(fma(scaled, p, kRound)) & ((1ull << 51) - 1);
  }
  __device__ __forceinline__ uint64_t weight(uint32_t key) const {
    return key >= alive ? weight_of(exponent(key)) : 0ull;
  }
  // The least key above -inf with a place below `bound` > 0, for a converged warp: around where the bound's logit
  // should be, then by a 32-way search.
  __device__ __forceinline__ uint32_t least_key(float bound) const {
    uint32_t lo = kNegInf, hi = top;  // lo fails, hi holds
    const int lane = threadIdx.x & 31;
    auto narrow = [&](uint32_t k) {
      const bool holds = place(k) < bound;
      hi = min(hi, __reduce_min_sync(0xffffffffu, holds ? k : top));
      lo = max(lo, __reduce_max_sync(0xffffffffu, holds ? kNegInf : k));
    };
    const float at = top_value - bound / bin_scale;
    if (hi - lo > 32 && fabsf(at) < INFINITY) {
      const uint32_t g = key_of(at), d = 1u << (2 * (lane & 15));
      const uint32_t k = lane < 16 ? (g > kNegInf + d ? g - d : kNegInf + 1) : (top - kNegInf > d && g < top - d ? g + d : top);
      narrow(min(max(k, kNegInf + 1), top));
    }
    while (hi - lo > 1) narrow(lo + 1 + (uint32_t)(((uint64_t)(hi - lo - 1) * lane) >> 5));
    return hi;
  }
  __device__ __forceinline__ bool inside(uint32_t key, uint32_t idx) const {
    return key > cut_key || (key == cut_key && idx <= cut_idx);
  }
};

struct Cluster {
  Shared& sh;
  Hist& hist;
  int rank, size, turn;
  __device__ __forceinline__ uint32_t at(const void* p, int r) const { return mapa_shared(smem_u32(p), r); }
  // Every CTA sends (a, b) to all; on return slots() holds all of them. All threads call.
  __device__ __forceinline__ const uint64_t (*exchange(uint64_t a, uint64_t b))[2] {
    const int t = turn;
    turn ^= 1;
    __syncthreads();
    if ((int)threadIdx.x < size) {
      const uint32_t d = at(&sh.slot[t][rank][0], threadIdx.x);
      st_cluster_u64(d, a);
      st_cluster_u64(d + 8, b);
    }
    cluster_barrier();
    return sh.slot[t];
  }
};

// Block sum; every thread gets it.
__device__ __forceinline__ uint64_t block_sum(Shared& sh, uint64_t a) {
#pragma unroll
  for (int o = 16; o; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh.warp[threadIdx.x >> 5][0] = a;
  __syncthreads();
  a = 0;
  for (int i = 0; i < kWarps; ++i) a += sh.warp[i][0];
  return a;
}
// Exclusive block scan of a value in thread order; the total in *total.
__device__ __forceinline__ uint64_t block_scan(Shared& sh, uint64_t v, uint64_t* total) {
  uint64_t inc = v;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t n = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += n;
  }
  __syncthreads();
  if (lane == 31) sh.warp[w][0] = inc;
  __syncthreads();
  uint64_t before = 0, all = 0;
  for (int i = 0; i < kWarps; ++i) {
    if (i < w) before += sh.warp[i][0];
    all += sh.warp[i][0];
  }
  *total = all;
  return before + inc - v;
}

// fn(key, position in the chunk) for this thread's keys, four neighbours at a time
template <typename Fn>
__device__ __forceinline__ void each_key(const uint32_t* keys, int n4, Fn fn) {
#pragma unroll 2
  for (int i = threadIdx.x; i < n4; i += kThreads) {
    const uint4 k = reinterpret_cast<const uint4*>(keys)[i];
    fn(k.x, 4 * i);
    fn(k.y, 4 * i + 1);
    fn(k.z, 4 * i + 2);
    fn(k.w, 4 * i + 3);
  }
}

__device__ __forceinline__ void clear_hist(Hist& h) {
  uint4* w = reinterpret_cast<uint4*>(&h);
  for (int b = threadIdx.x; b < (int)(sizeof(Hist) / 16); b += kThreads) w[b] = make_uint4(0, 0, 0, 0);
}

// Publishes this CTA's histogram: the sums of its groups of 32 bins go to every CTA (reading whole histograms
// through the cluster costs 16 CTAs 7 us). All threads call it; ends with a barrier of the cluster.
__device__ __forceinline__ void publish(const Cluster& c) {
  __syncthreads();
  const int lane = threadIdx.x & 31;
  for (int g = threadIdx.x >> 5; g < kBins / 32; g += kWarps) {
    uint64_t v = c.hist.bin[g * 32 + lane];
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (lane < c.size) st_cluster_u64(c.at(&c.sh.group[c.rank][g], lane), v);
  }
  cluster_barrier();
}
// The sum of all published bins.
__device__ __forceinline__ uint64_t published(const Cluster& c) {
  uint64_t v = 0;
  if (threadIdx.x < kBins / 32)
    for (int r = 0; r < c.size; ++r) v += c.sh.group[r][threadIdx.x];
  return block_sum(c.sh, v);
}

// The bin in which the running value (from the largest logits on, `before` ahead of the first) reaches the goal,
// over the whole cluster's histograms: every CTA finds it for itself. The goal is within reach.
struct Found {
  int bin;
  uint64_t before, value;
};
__device__ __forceinline__ Found find_bin(const Cluster& c, uint64_t before, uint64_t goal) {
  static_assert(kBins / 32 <= kThreads);
  Shared& sh = c.sh;
  uint64_t v = 0, all;
  if (threadIdx.x < kBins / 32)
    for (int r = 0; r < c.size; ++r) v += sh.group[r][threadIdx.x];
  const uint64_t run = before + block_scan(sh, v, &all);
  if (run < goal && goal <= run + v) {
    sh.found[0] = run;
    sh.found_bin = threadIdx.x;
  }
  __syncthreads();
  if (threadIdx.x < 32) {  // the group's bins, a lane each
    const int b = sh.found_bin * 32 + threadIdx.x;
    uint64_t w = 0, inc;
#pragma unroll 4
    for (int r = 0; r < c.size; ++r) w += ld_cluster_u64(c.at(&c.hist.bin[b], r));
    inc = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t up = __shfl_up_sync(0xffffffffu, inc, o);
      if ((int)threadIdx.x >= o) inc += up;
    }
    const uint64_t from = sh.found[0] + inc - w;
    __syncwarp();
    if (from < goal && goal <= from + w) {
      sh.found[0] = from;
      sh.found[1] = w;
      sh.found_bin = b;
    }
  }
  __syncthreads();
  const Found f{sh.found_bin, sh.found[0], sh.found[1]};
  __syncthreads();
  return f;
}

__device__ __forceinline__ uint64_t goal_of_u(float uf, uint64_t z) {
  const double u = (double)uf, g = u > 0.0 ? u * (double)z : 0.0;
  return g < (double)z ? min((uint64_t)g, z - 1) : z - 1;
}
__device__ __forceinline__ void put_token(const SampleParams& p, int b, const Row& row, uint32_t key, uint32_t idx,
                                          uint64_t z) {
  p.tok[b] = (int32_t)idx;
  if (p.tok2) p.tok2[b] = (int32_t)idx;
  if (p.logprob) p.logprob[b] = (float)(row.exponent(key) - log((double)z / (double)(1ull << row.S)));
}

// The share of `total` that top-p keeps, rounded up: the prefix ends with the element that reaches it.
__device__ __forceinline__ uint64_t goal_of_p(float p, uint64_t total) {
  const double g = ceil((double)p * (double)total);
  return g < 1.0 ? 1ull : (uint64_t)g < total ? (uint64_t)g : total;
}

// The cluster's first CTA finishes a row from its list of candidates, which holds
// every element down to the cut: one per thread, against all others. k: elements to
// keep; goal: mass to reach, or with RANKED top_p of the first k's.
template <bool RANKED>
__device__ void finish(Shared& sh, const SampleParams& p, int b, const Row& row, uint64_t k, uint64_t goal, float top_p) {
  const int tid = threadIdx.x, n = (int)sh.ncand;
  // 2^lg threads per candidate share the comparisons
  int lg = 0;
  while (lg < 5 && (n << (lg + 1)) <= kThreads) ++lg;
  const int i = tid >> lg, part = tid & ((1 << lg) - 1), step = 1 << lg;
  const bool mine = i < n, lead = mine && part == 0;
  const uint32_t key = mine ? sh.ckey[i] : 0, idx = mine ? sh.cidx[i] : 0;
  const uint64_t w = mine ? row.weight(key) : 0;
  if (lead) sh.cmass[i] = w;
  __syncthreads();
  uint64_t before = 0;
  uint32_t rank = 0;
  if (((tid & ~31) >> lg) < n) {
#pragma unroll 4
    for (int j = part; j < n; j += step) {
      const uint32_t kj = sh.ckey[j], xj = sh.cidx[j];
      const uint64_t wj = sh.cmass[j];
      const bool ahead = kj > key || (kj == key && xj < idx);
      before += ahead ? wj : 0;
      rank += ahead;
    }
    for (int o = step >> 1; o; o >>= 1) {
      before += __shfl_xor_sync(0xffffffffu, before, o);
      rank += __shfl_xor_sync(0xffffffffu, rank, o);
    }
  }
  bool keep = mine && w > 0;
  if (RANKED) {
    keep = keep && rank < k;
    const uint64_t zk = block_sum(sh, keep && lead ? w : 0);
    goal = top_p < 1.0f ? goal_of_p(top_p, zk) : zk;
  }
  keep = keep && before < goal && row.exponent(key) >= row.min_e;
  __syncthreads();
  if (lead) sh.cmass[i] = keep ? w : 0;
  const uint64_t z = block_sum(sh, keep && lead ? w : 0);  // (its barriers publish cmass)
  const uint64_t g = goal_of_u(p.u[b], z);
  uint64_t run = 0;
  if (((tid & ~31) >> lg) < n) {
#pragma unroll 4
    for (int j = part; j < n; j += step) {
      const uint32_t xj = sh.cidx[j];
      const uint64_t wj = sh.cmass[j];
      run += xj < idx ? wj : 0;
    }
    for (int o = step >> 1; o; o >>= 1) run += __shfl_xor_sync(0xffffffffu, run, o);
  }
  if (keep && lead && run <= g && g < run + w) put_token(p, b, row, key, idx, z);
}

// Sends this CTA's elements with keys in [lo, hi] (inside the cut) to the first CTA's list. Ends with a barrier of
// the cluster; returns how many there were in all: at most kCand of them are in the list.
__device__ __forceinline__ uint32_t gather(const Cluster& c, const Row& row, const uint32_t* keys, int n4, uint32_t idx0,
                                           uint32_t lo, uint32_t hi, bool skip) {
  const uint32_t n_at = c.at(&c.sh.ncand, 0), key_at = c.at(c.sh.ckey, 0), idx_at = c.at(c.sh.cidx, 0);
  if (!skip)
    each_key(keys, n4, [&](uint32_t key, int i) {
      if (key < lo || key > hi || !row.inside(key, idx0 + i)) return;
      const uint32_t at = atom_cluster_inc(n_at);
      if (at >= (uint32_t)kCand) return;
      st_cluster_b32(key_at + at * 4, key);
      st_cluster_b32(idx_at + at * 4, idx0 + i);
    });
  cluster_barrier();
  return ld_cluster_u32(n_at);
}

// The first CTA works, and leaves only after every CTA of the cluster has read its shared memory for the last time.
template <typename Fn>
__device__ __forceinline__ void last_read(const Cluster& c, Fn work) {
  __syncwarp();
  cluster_arrive_release();
  if (c.rank == 0) work();
  __syncwarp();
  cluster_wait_acquire();
}

// Top-k from the threads' largest logits (see the top): true when the row is
// finished, false when there are too few or too many for it. All threads of the
// cluster call it.
__device__ bool top_of_threads(Cluster& c, const SampleParams& p, int b, Row& row, const uint32_t* keys, int n4,
                               uint32_t idx0, uint32_t largest, uint64_t k, float top_p) {
  if (largest >= row.alive) atomicAdd(&c.hist.bin[(int)row.place(largest)], 1ull);
  if (threadIdx.x == 0) c.sh.ncand = 0;
  publish(c);
  bool done = false;
  if (published(c) >= k) {
    const Found f = find_bin(c, 0, k);
    if (f.before + f.value <= (uint64_t)kCand) {
      const uint32_t lo = row.least_key((float)(f.bin + 1));
      done = gather(c, row, keys, n4, idx0, lo, 0xffffffffu, largest < lo) <= (uint32_t)kCand;
    }
  }
  if (done) {
    last_read(c, [&] { finish<true>(c.sh, p, b, row, k, 0, top_p); });
    return true;
  }
  cluster_barrier();  // the histograms and the list have been read
  clear_hist(c.hist);
  __syncthreads();
  return false;
}

// The cut of the shortest prefix whose value (its count: top-k; its mass: top-p)
// reaches a goal: k, or top_p of the mass inside the present cut. True when the row
// is finished. The histogram is clear on entry. All threads of the cluster call it,
// and every branch on the way to a barrier is the same for all of them.
template <bool MASS>
__device__ bool select(Cluster& c, const SampleParams& p, int row_b, Row& row, const uint32_t* keys, int n4,
                       uint32_t idx0, uint64_t k, float top_p) {
  Shared& sh = c.sh;
  const int tid = threadIdx.x;
  uint64_t before = 0, goal = 0;              // the value of what lies above the range; the goal
  uint32_t lo = row.alive, hi = 0xffffffffu;  // keys of the range, inclusive
  int shift = 0;
  bool first = true;  // the first histogram is over Row::place, the others over the bits of the keys
  for (int pass = 0; pass < 6; ++pass) {  // at most 4 are needed: 2048 bins, then 11 bits of the key each
    each_key(keys, n4, [&](uint32_t key, int i) {
      if (key < lo || key > hi || !row.inside(key, idx0 + i)) return;
      const int b = first ? (int)row.place(key) : (int)((hi - key) >> shift);
      const uint64_t v = MASS ? row.weight_of(row.exponent(key)) : 1ull;
      if (v) atomicAdd(&c.hist.bin[b], (unsigned long long)v);
    });
    if (tid == 0) sh.ncand = 0;
    publish(c);
    if (first) {
      const uint64_t total = published(c);
      goal = MASS ? goal_of_p(top_p, total) : k;
      if (goal > total || (!MASS && goal == total)) {  // nothing to cut off
        cluster_barrier();                             // (the sums are read before they are written again)
        return false;
      }
    }
    const Found f = find_bin(c, before, goal);
    before = f.before;
    uint32_t klo, khi;  // the keys of its bin
    if (first) {
      klo = row.least_key((float)(f.bin + 1));
      khi = f.bin ? row.least_key((float)f.bin) - 1 : 0xffffffffu;
    } else {
      khi = hi - ((uint32_t)f.bin << shift);
      klo = khi - lo > (1u << shift) - 1 ? khi - ((1u << shift) - 1) : lo;
    }
    // how many elements there are: counted, or bounded by the least and the greatest mass that they may have
    const uint64_t w_lo = MASS ? row.weight(klo) : 1, w_hi = MASS ? row.weight(min(khi, row.top)) : 1;
    const bool down = first && before + f.value <= kCand * w_lo;
    if (down || f.value <= kCand * w_hi) {
      const uint32_t m = gather(c, row, keys, n4, idx0, klo, down ? 0xffffffffu : khi, false);
      if (m <= (uint32_t)kCand) {
        if (down) {
          last_read(c, [&] { finish<!MASS>(sh, p, row_b, row, k, goal, top_p); });
          return true;
        }
        if (c.rank == 0) {
          if (tid < (int)m) sh.cmass[tid] = MASS ? row.weight(sh.ckey[tid]) : 1ull;
          if (tid == 0) sh.found[0] = sh.found[1] = 0;
          __syncthreads();
          if (tid < (int)m) {
            const uint32_t ki = sh.ckey[tid], xi = sh.cidx[tid];
            uint64_t v = before;
#pragma unroll 4
            for (int j = 0; j < (int)m; ++j) {
              const uint32_t kj = sh.ckey[j], xj = sh.cidx[j];
              const uint64_t wj = sh.cmass[j];
              v += kj > ki || (kj == ki && xj < xi) ? wj : 0;
            }
            if (v < goal && goal <= v + sh.cmass[tid]) {
              sh.found[0] = ki;
              sh.found[1] = xi;
            }
          }
          __syncthreads();
        }
        const auto cut = c.exchange(sh.found[0], sh.found[1]);
        row.cut_key = (uint32_t)cut[0][0];
        row.cut_idx = (uint32_t)cut[0][1];
        return false;
      }
    }
    if (klo == min(khi, row.top)) {
      // many equal keys: the goal's place among them, in index order
      const uint64_t g = w_lo, need = (goal - before + g - 1) / g;  // ties to keep, >= 1
      uint64_t ties = 0;
      const int blk = (n4 + kThreads - 1) / kThreads * 4, i0 = min(4 * n4, tid * blk), i1 = min(4 * n4, i0 + blk);
      for (int i = i0; i < i1; ++i) ties += keys[i] == klo && row.inside(klo, idx0 + i);
      uint64_t all;
      const uint64_t tpre = block_scan(sh, ties, &all);
      const auto tslots = c.exchange(all, 0);
      uint64_t tb = tpre;
      for (int r = 0; r < c.rank; ++r) tb += tslots[r][0];
      if (tid == 0) sh.found[0] = ~0ull;
      __syncthreads();
      if (tb < need && need <= tb + ties) {
        for (int i = i0; i < i1; ++i)
          if (keys[i] == klo && row.inside(klo, idx0 + i) && ++tb == need) sh.found[0] = idx0 + i;
      }
      __syncthreads();
      const auto cut = c.exchange(sh.found[0], 0);
      for (int r = 0; r < c.size; ++r)
        if (cut[r][0] != ~0ull) {
          row.cut_key = klo;
          row.cut_idx = (uint32_t)cut[r][0];
        }
      return false;
    }
    // many elements of unlike keys: another histogram over the bin's keys
    cluster_barrier();  // every CTA has read the histograms
    lo = klo;
    hi = min(khi, row.top);
    first = false;
    shift = max(0, 32 - __clz(hi - lo) - 11);  // hi - lo < 2^(32 - clz)
    clear_hist(c.hist);
    __syncthreads();
  }
  return false;
}

__global__ void __launch_bounds__(kThreads) sample_kernel(const __grid_constant__ SampleParams p) {
  extern __shared__ __align__(16) uint32_t keys[];  // [chunk], then the histograms when there are top_k or top_p
  __shared__ Shared sh;
  uint32_t size;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(size));
  Cluster c{sh, *reinterpret_cast<Hist*>(keys + p.chunk), (int)cluster_ctarank(), (int)size, 0};
  const int b = blockIdx.x / size, tid = threadIdx.x, n4 = p.chunk / 4;
  const uint32_t idx0 = c.rank * p.chunk;
  if (tid < 64) sh.exp2_64[tid] = exp2(tid / 64.0);
  if (p.top_k || p.top_p) clear_hist(c.hist);
  pdl_launch_dependents();
  pdl_wait();
  // the chunk's keys, and its largest with the lowest index
  const float T = p.temp ? p.temp[b] : 1.0f;
  const int k = p.top_k ? p.top_k[b] : 0;
  const float tp = p.top_p ? p.top_p[b] : 1.0f;
  uint64_t best = 0;
  auto put = [&](int i, const float (&v)[4], int n) {  // four neighbours, n of them logits
    uint32_t q[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      q[e] = e < n ? key_of(v[e]) : 0;
      const uint64_t cand = ((uint64_t)q[e] << 32) | (uint32_t)~(idx0 + 4 * i + e);
      if (e < n && cand > best) best = cand;
    }
    reinterpret_cast<uint4*>(keys)[i] = make_uint4(q[0], q[1], q[2], q[3]);
  };
  auto load = [&](auto type) {
    using T_ = decltype(type);
    const T_* x = static_cast<const T_*>(p.x) + (int64_t)b * p.ld + idx0;
    const int n = min((int)max((int64_t)0, (int64_t)p.V - idx0), p.chunk);
    // rows that begin off a 4-logit boundary are read one by one
    const bool whole = (reinterpret_cast<uintptr_t>(static_cast<const T_*>(p.x) + (int64_t)b * p.ld) % (4 * sizeof(T_))) == 0;
    const int full = whole ? n / 4 : 0;
    int i = tid;
#pragma unroll 4
    for (; i < full; i += kThreads) {
      Pack<T_, 4> w;
      w.load(x + 4 * i);
      const float v[4] = {w.get(0), w.get(1), w.get(2), w.get(3)};
      put(i, v, 4);
    }
    for (; i < n4; i += kThreads) {
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = 4 * i + e < n ? to_f32(x[4 * i + e]) : 0.0f;
      put(i, v, n - 4 * i);
    }
  };
  if (p.type == BTF_F32) load(0.0f);
  else if (p.type == BTF_F16) load(__half());
  else load(__nv_bfloat16());
  const uint32_t largest = (uint32_t)(best >> 32);  // this thread's
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const uint64_t q = __shfl_xor_sync(0xffffffffu, best, o);
    best = q > best ? q : best;
  }
  if ((tid & 31) == 0) sh.warp[tid >> 5][0] = best;
  __syncthreads();
  for (int i = 0; i < kWarps; ++i) best = sh.warp[i][0] > best ? sh.warp[i][0] : best;
  {
    const auto s = c.exchange(best, 0);
    for (int r = 0; r < c.size; ++r) best = s[r][0] > best ? s[r][0] : best;
  }
  Row row;
  row.top = (uint32_t)(best >> 32);
  const uint32_t top_idx = ~(uint32_t)best;
  const bool none = row.top <= kNegInf;
  if (none || !(T > 0.0f)) {  // nothing to draw from, or greedy
    if (c.rank == 0 && tid == 0) {
      const int32_t t = none ? 0 : (int32_t)top_idx;
      p.tok[b] = t;
      if (p.tok2) p.tok2[b] = t;
      if (p.logprob) p.logprob[b] = none ? __uint_as_float(0x7fc00000u) : 0.0f;
    }
    return;
  }
  row.top_value = key_value(row.top);
  row.m = (double)row.top_value;
  row.inv_t = 1.0 / (double)T;
  row.bin_scale = (float)kBins / kSpan / T;
  row.S = p.S;
  row.cut_key = 0;
  row.cut_idx = 0xffffffffu;
  row.table = sh.exp2_64;
  row.alive = row.least_key((float)kBins);
  row.min_e = -INFINITY;
  uint32_t least = row.alive;  // keys below are not kept
  {
    const float mp = p.min_p ? p.min_p[b] : 0.0f;
    if (mp > 0.0f) {
      row.min_e = fmin(log((double)mp), 0.0);
      // place() is within 2^-22 of the exact one, relative
      const float bound = (float)(-row.min_e * (kBins / kSpan)) * (1.0f + 0x1p-20f) + 0x1p-20f;
      if (bound < (float)kBins) least = row.least_key(bound);
    }
  }
  const bool ks = k > 0 && k < p.V;
  if (ks) {
    // (more than the ranking can hold needs no try)
    if (k <= kCand && top_of_threads(c, p, b, row, keys, n4, idx0, largest, (uint64_t)k, tp)) return;
    if (select<false>(c, p, b, row, keys, n4, idx0, (uint64_t)k, tp)) return;
  }
  if (tp < 1.0f) {
    if (ks) {
      __syncthreads();
      clear_hist(c.hist);
      __syncthreads();
    }
    if (select<true>(c, p, b, row, keys, n4, idx0, 0, tp)) return;
  }
  least = max(least, row.cut_key);
  // running masses in index order: a warp owns a contiguous block
  const int lane = tid & 31, w = tid >> 5, blk = n4 / kWarps, w0 = w * blk;  // in fours of keys
  auto kept = [&](uint32_t key, int i) -> uint64_t {
    if (key < least || !row.inside(key, idx0 + i)) return 0ull;
    const double e = row.exponent(key);
    return e >= row.min_e ? row.weight_of(e) : 0ull;
  };
  uint64_t mine = 0;
#pragma unroll 2
  for (int i = w0 + lane; i < w0 + blk; i += 32) {
    const uint4 q = reinterpret_cast<const uint4*>(keys)[i];
    mine += kept(q.x, 4 * i) + kept(q.y, 4 * i + 1) + kept(q.z, 4 * i + 2) + kept(q.w, 4 * i + 3);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  __syncthreads();
  if (lane == 0) sh.warp[w][0] = mine;
  __syncthreads();
  uint64_t cta = 0, pre = 0;
  for (int i = 0; i < kWarps; ++i) {
    if (i < w) pre += sh.warp[i][0];
    cta += sh.warp[i][0];
  }
  const auto s = c.exchange(cta, 0);
  uint64_t z = 0;
  for (int r = 0; r < c.size; ++r) {
    if (r < c.rank) pre += s[r][0];
    z += s[r][0];
  }
  const uint64_t goal = goal_of_u(p.u[b], z);
  if (pre <= goal && goal < pre + mine) {
    // the warp that holds the token walks its block
    for (int i0 = w0; i0 < w0 + blk; i0 += 32) {
      const int i = i0 + lane;
      const uint4 q = i < w0 + blk ? reinterpret_cast<const uint4*>(keys)[i] : make_uint4(0, 0, 0, 0);
      const uint32_t key[4] = {q.x, q.y, q.z, q.w};
      uint64_t v[4], inc = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = kept(key[e], 4 * i + e), inc += v[e];
      const uint64_t four = inc;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint64_t up = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += up;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, pre + inc > goal);
      if (hit) {
        if (lane == __ffs(hit) - 1) {
          uint64_t run = pre + inc - four;
          bool done = false;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            run += v[e];
            if (!done && run > goal) {
              put_token(p, b, row, key[e], idx0 + 4 * i + e, z);
              done = true;
            }
          }
        }
        break;
      }
      pre += __shfl_sync(0xffffffffu, inc, 31);
    }
  }
}

}  // namespace

int sample_setup(DeviceInfo& d) {
  constexpr int kMost = BTF_SAMPLE_MAX_V / kMaxCluster * 4 + (int)sizeof(Hist);  // the largest chunk's keys
  if (kMost + (int)sizeof(Shared) + 1024 > d.optin_smem)
    return fail(BTF_ERR_UNSUPPORTED, "sample_kernel needs %d bytes of shared memory", kMost + (int)sizeof(Shared));
  cudaError_t e = cudaFuncSetAttribute(sample_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(sample_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  return e == cudaSuccess ? BTF_OK : cuda_fail(e, "sample_kernel attributes");
}

cudaError_t launch_sample(const SampleArgs& a, cudaStream_t st) {
  SampleParams p{a.logits, a.ld, a.type, a.V, 0, 62, a.u, a.temperature, a.top_p, a.min_p, a.top_k, a.tokens, a.tokens2,
                 a.logprobs};
  int lg = 0;
  while ((1ll << lg) < a.V) ++lg;
  p.S = std::min(44, 62 - lg);
  // a CTA per about 16384 logits: its keys stay in shared memory
  int size = 1;
  while (size < kMaxCluster && (a.V + size - 1) / size > 16384) size *= 2;
  constexpr int kStep = 4 * kThreads;
  p.chunk = ((a.V + size - 1) / size + kStep - 1) / kStep * kStep;
  const size_t smem = (size_t)p.chunk * 4 + (a.top_k || a.top_p ? sizeof(Hist) : 0);
  return launch_pdl_cluster(sample_kernel, dim3((unsigned)(a.B * size)), dim3(kThreads), smem, st, size, p);
}

}  // namespace btf

using namespace btf;

extern "C" {

int btf_sample(const void* logits, int type, int64_t ld, int B, int V, const float* u, const float* temperature,
               const int32_t* top_k, const float* top_p, const float* min_p, int32_t* tokens, float* logprobs,
               void* stream) {
  if (B < 0 || V < 1 || V > BTF_SAMPLE_MAX_V || ld < V)
    return fail(BTF_ERR_ARG, "btf_sample: need B >= 0, 1 <= V <= %d and ld >= V (B %d, V %d, ld %lld)", BTF_SAMPLE_MAX_V,
                B, V, (long long)ld);
  if (!elem_type_ok(type)) return fail(BTF_ERR_ARG, "btf_sample: unknown element type %d", type);
  if (B == 0) return BTF_OK;
  if (B > (1 << 24)) return fail(BTF_ERR_ARG, "btf_sample: at most 2^24 rows");
  if (!logits || !u || !tokens) return fail(BTF_ERR_ARG, "btf_sample: null logits, u or tokens");
  if (reinterpret_cast<uintptr_t>(logits) % elem_bytes(type))
    return fail(BTF_ERR_ARG, "btf_sample: logits are not aligned to their type");
  if (!current_device()) return BTF_ERR_STATE;
  const SampleArgs a{logits, type, ld, B, V, u, temperature, top_k, top_p, min_p, tokens, nullptr, logprobs};
  const cudaError_t e = launch_sample(a, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? BTF_OK : cuda_fail(e, "btf_sample");
}

}  // extern "C"
