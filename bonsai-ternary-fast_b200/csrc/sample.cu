// Sampling from given random numbers (btf_sample): temperature, top-k, top-p and
// min-p on one row of logits per thread-block cluster, whose shared memory holds the
// row: the logits are read once.
//
// All three filters keep a prefix of the order (logit descending, index
// ascending), so nothing is sorted: a cut (key, index) in that order plus a bound on
// the exponent is the kept set. A cut is found by a histogram over 2048 bins of
// (max - l) / T. When the bins down to the cut's hold few elements (a top-k of 50, a
// peaked nucleus), those go to the cluster's first CTA, which ranks them exactly and
// finishes the row. Else the elements of the cut's own bin are ranked (or, when there
// are many, split further by the bits of their keys), and the token comes from a
// walk over running masses in index order, each CTA over its own part of the row.
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
  uint64_t total[kMaxCluster];       // each CTA's part of a histogram's total
  uint64_t warp[kWarps][2];
  uint64_t found[2];
  double exp2_64[64];  // 2^(i / 64)
  uint64_t cmass[kCand];
  uint32_t ckey[kCand], cidx[kCand];
  uint32_t ncand;
};
// The histograms: counts, and the bins' masses in 16-bit limbs (a CTA holds at most 2^16 elements).
struct Hist {
  uint32_t cnt[kBins];
  uint32_t mass[3][kBins];
};

// One row's state, the same in every thread of the cluster.
struct Row {
  uint32_t top;     // key of the largest logit
  float top_value;
  double m, inv_t;  // the largest logit and 1 / T
  float bin_scale;
  double min_e;     // min-p: exponents below are dropped
  float min_bin;    // a bound on their place among the bins, with room for rounding
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
    return place(key) < (float)kBins ? weight_of(exponent(key)) : 0ull;
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

__device__ __forceinline__ void clear_hist(Hist& h, bool mass) {
  for (int b = threadIdx.x; b < kBins; b += kThreads) {
    h.cnt[b] = 0;
    if (mass) h.mass[0][b] = h.mass[1][b] = h.mass[2][b] = 0;
  }
}

// A bin's value over the whole cluster: its count, or its mass.
template <bool MASS>
__device__ __forceinline__ uint64_t bin_value(const Cluster& c, int b) {
  uint64_t v = 0;
#pragma unroll 4
  for (int r = 0; r < c.size; ++r) {
    const uint32_t base = c.at(&c.hist, r) + b * 4;
    if (MASS)
      v += (uint64_t)ld_cluster_u32(base + 4 * kBins) + ((uint64_t)ld_cluster_u32(base + 8 * kBins) << 16) +
           ((uint64_t)ld_cluster_u32(base + 12 * kBins) << 32);
    else
      v += ld_cluster_u32(base);
  }
  return v;
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
  const bool mine = tid < n;
  const uint32_t key = mine ? sh.ckey[tid] : 0, idx = mine ? sh.cidx[tid] : 0;
  const uint64_t w = mine ? row.weight(key) : 0;
  if (mine) sh.cmass[tid] = w;
  __syncthreads();
  uint64_t before = 0;
  uint32_t rank = 0;
#pragma unroll 4
  for (int j = 0; j < n; ++j) {
    const uint32_t kj = sh.ckey[j];
    if (kj > key || (kj == key && sh.cidx[j] < idx)) {
      before += sh.cmass[j];
      ++rank;
    }
  }
  bool keep = mine && w > 0;
  if (RANKED) {
    keep = keep && rank < k;
    const uint64_t zk = block_sum(sh, keep ? w : 0);
    goal = top_p < 1.0f ? goal_of_p(top_p, zk) : zk;
  }
  keep = keep && before < goal && row.exponent(key) >= row.min_e;
  __syncthreads();
  if (mine) sh.cmass[tid] = keep ? w : 0;
  const uint64_t z = block_sum(sh, keep ? w : 0);  // (its barriers publish cmass)
  const uint64_t g = goal_of_u(p.u[b], z);
  uint64_t run = 0;
#pragma unroll 4
  for (int j = 0; j < n; ++j)
    if (sh.cidx[j] < idx) run += sh.cmass[j];
  if (keep && run <= g && g < run + w) put_token(p, b, row, key, idx, z);
}

// The cut of the shortest prefix whose value (its count: top-k; its mass: top-p)
// reaches a goal: k, or top_p of the mass inside the present cut. True when the row
// is finished. All threads of the cluster call it, and every branch on the way to a
// barrier is the same for all of them.
template <bool MASS>
__device__ bool select(Cluster& c, const SampleParams& p, int row_b, Row& row, const uint32_t* keys, int n4,
                       uint32_t idx0, uint64_t k, float top_p) {
  Shared& sh = c.sh;
  Hist& h = c.hist;
  const int tid = threadIdx.x;
  uint64_t before = 0, goal = 0;      // the value of what lies above the range; the goal
  uint32_t lo = 0, hi = 0xffffffffu;  // keys of the range, inclusive
  int shift = 0;
  bool first = true;  // the first histogram is over Row::place (it was cleared by the caller)
  // bin of an element of the range, or -1
  auto bin_of = [&](uint32_t key, uint32_t idx) -> int {
    const float at = row.place(key);
    if (!(at < (float)kBins) || !row.inside(key, idx)) return -1;
    if (first) return (int)at;
    return key < lo || key > hi ? -1 : (int)((hi - key) >> shift);
  };
  for (int pass = 0; pass < 6; ++pass) {  // at most 4 are needed: 2048 bins, then 11 bits of the key each
    uint64_t sum = 0;
    each_key(keys, n4, [&](uint32_t key, int i) {
      const int b = bin_of(key, idx0 + i);
      if (b < 0) return;
      atomicAdd(&h.cnt[b], 1u);
      if (MASS) {
        const uint64_t w = row.weight_of(row.exponent(key));
        atomicAdd(&h.mass[0][b], (uint32_t)(w & 0xffffu));
        atomicAdd(&h.mass[1][b], (uint32_t)((w >> 16) & 0xffffu));
        atomicAdd(&h.mass[2][b], (uint32_t)(w >> 32));
        sum += w;
      } else {
        ++sum;
      }
    });
    if (first) {
      sum = block_sum(sh, sum);
      if (tid < c.size) st_cluster_u64(c.at(&sh.total[c.rank], tid), sum);
      if (tid == 0) sh.ncand = 0;
    }
    __syncthreads();
    cluster_barrier();
    if (first) {
      uint64_t total = 0;
      for (int r = 0; r < c.size; ++r) total += sh.total[r];
      goal = MASS ? goal_of_p(top_p, total) : k;
      if (goal > total || (!MASS && goal == total)) {  // nothing to cut off
        cluster_barrier();  // (sh.total is read before it is written again)
        return false;
      }
    }
    // every CTA finds the bin for itself, a thread per bin from the largest on
    int bin = 0;
    uint32_t count = 0;
    for (int b0 = 0;; b0 += kThreads) {
      const uint64_t v = bin_value<MASS>(c, b0 + tid);
      uint64_t all;
      const uint64_t pre = before + block_scan(sh, v, &all);
      if (pre < goal && goal <= pre + v) {
        sh.found[0] = ((uint64_t)(b0 + tid) << 32) | (uint32_t)bin_value<false>(c, b0 + tid);
        sh.found[1] = pre;
      }
      __syncthreads();
      if (goal <= before + all || b0 + kThreads >= kBins) break;
      before += all;
    }
    bin = (int)(sh.found[0] >> 32);
    count = (uint32_t)sh.found[0];
    before = sh.found[1];
    // few elements down to this bin: the first CTA ranks them and finishes the row
    uint64_t down = ~0ull;
    if (first) {
      if (!MASS) {
        down = before + count;
      } else {
        uint64_t part = 0;
        for (int b = tid; b < bin; b += kThreads) part += bin_value<false>(c, b);
        down = block_sum(sh, part) + count;
      }
    }
    if (down <= (uint64_t)kCand || count <= (uint32_t)kCand) {
      const bool all = down <= (uint64_t)kCand;
      const uint32_t n_at = c.at(&sh.ncand, 0), key_at = c.at(sh.ckey, 0), idx_at = c.at(sh.cidx, 0);
      each_key(keys, n4, [&](uint32_t key, int i) {
        const int b = bin_of(key, idx0 + i);
        if (b < 0 || (all ? b > bin : b != bin)) return;
        const uint32_t at = atom_cluster_inc(n_at);
        if (at >= (uint32_t)kCand) return;
        st_cluster_b32(key_at + at * 4, key);
        st_cluster_b32(idx_at + at * 4, idx0 + i);
      });
      cluster_barrier();
      if (all) {
        if (c.rank == 0) finish<!MASS>(sh, p, row_b, row, k, goal, top_p);
        return true;
      }
      if (c.rank == 0) {
        const int m = (int)min(sh.ncand, (uint32_t)kCand);
        if (tid < m) sh.cmass[tid] = MASS ? row.weight(sh.ckey[tid]) : 1ull;
        if (tid == 0) sh.found[0] = sh.found[1] = 0;
        __syncthreads();
        if (tid < m) {
          const uint32_t ki = sh.ckey[tid], xi = sh.cidx[tid];
          uint64_t v = before;
#pragma unroll 4
          for (int j = 0; j < m; ++j) {
            const uint32_t kj = sh.ckey[j];
            if (kj > ki || (kj == ki && sh.cidx[j] < xi)) v += sh.cmass[j];
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
    if (!first && shift == 0) {
      // many equal keys: the goal's place among them, in index order
      const uint32_t key = hi - bin;
      const uint64_t g = MASS ? row.weight(key) : 1ull;
      const uint64_t need = (goal - before + g - 1) / g;  // ties to keep, >= 1
      uint64_t ties = 0;
      const int blk = (n4 + kThreads - 1) / kThreads * 4, i0 = min(4 * n4, tid * blk), i1 = min(4 * n4, i0 + blk);
      for (int i = i0; i < i1; ++i) ties += keys[i] == key && row.inside(key, idx0 + i);
      uint64_t all;
      const uint64_t tpre = block_scan(sh, ties, &all);
      const auto tslots = c.exchange(all, 0);
      uint64_t tb = tpre;
      for (int r = 0; r < c.rank; ++r) tb += tslots[r][0];
      if (tid == 0) sh.found[0] = ~0ull;
      __syncthreads();
      if (tb < need && need <= tb + ties) {
        for (int i = i0; i < i1; ++i)
          if (keys[i] == key && row.inside(key, idx0 + i) && ++tb == need) sh.found[0] = idx0 + i;
      }
      __syncthreads();
      const auto cut = c.exchange(sh.found[0], 0);
      for (int r = 0; r < c.size; ++r)
        if (cut[r][0] != ~0ull) {
          row.cut_key = key;
          row.cut_idx = (uint32_t)cut[r][0];
        }
      return false;
    }
    // many elements of unlike keys: another histogram over the range of the bin's keys
    if (first) {
      uint32_t kmin = 0xffffffffu, kmax = 0;
      each_key(keys, n4, [&](uint32_t key, int i) {
        if (bin_of(key, idx0 + i) == bin) kmin = min(kmin, key), kmax = max(kmax, key);
      });
      kmin = __reduce_min_sync(0xffffffffu, kmin);
      kmax = __reduce_max_sync(0xffffffffu, kmax);
      __syncthreads();
      if ((tid & 31) == 0) sh.warp[tid >> 5][0] = kmin, sh.warp[tid >> 5][1] = kmax;
      __syncthreads();
      for (int i = 0; i < kWarps; ++i)
        kmin = min(kmin, (uint32_t)sh.warp[i][0]), kmax = max(kmax, (uint32_t)sh.warp[i][1]);
      const auto ks = c.exchange(kmin, kmax);
      for (int r = 0; r < c.size; ++r) kmin = min(kmin, (uint32_t)ks[r][0]), kmax = max(kmax, (uint32_t)ks[r][1]);
      lo = kmin;
      hi = kmax;
      first = false;
    } else {
      const uint32_t top = hi - ((uint32_t)bin << shift), width = (1u << shift) - 1;
      hi = top;
      lo = top - lo > width ? top - width : lo;
      cluster_barrier();  // every CTA has read the histograms
    }
    const int bits = hi > lo ? 32 - __clz(hi - lo) : 0;  // hi - lo < 2^bits
    shift = max(0, bits - 11);
    clear_hist(h, MASS);
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
  if (p.top_k || p.top_p) clear_hist(c.hist, p.top_p != nullptr);
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
  row.min_e = -INFINITY;
  row.min_bin = (float)kBins;
  {
    const float mp = p.min_p ? p.min_p[b] : 0.0f;
    if (mp > 0.0f) {
      row.min_e = fmin(log((double)mp), 0.0);
      // place() is within 2^-22 of the exact one, relative
      row.min_bin = fminf(row.min_bin, (float)(-row.min_e * (kBins / kSpan)) * (1.0f + 0x1p-20f) + 0x1p-20f);
    }
  }
  if (k > 0 && k < p.V && select<false>(c, p, b, row, keys, n4, idx0, (uint64_t)k, tp)) return;
  if (tp < 1.0f) {
    if (k > 0 && k < p.V) {
      __syncthreads();
      clear_hist(c.hist, true);
      __syncthreads();
    }
    if (select<true>(c, p, b, row, keys, n4, idx0, 0, tp)) return;
  }
  // running masses in index order: a warp owns a contiguous block
  const int lane = tid & 31, w = tid >> 5, blk = n4 / kWarps, w0 = w * blk;  // in fours of keys
  auto kept = [&](uint32_t key, int i) -> uint64_t {
    if (!(row.place(key) < row.min_bin) || !row.inside(key, idx0 + i)) return 0ull;
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
