// Sampling from given random numbers (btf_sample): temperature, top-k, top-p and
// min-p on one row of logits per thread-block cluster.
//
// All three filters keep a prefix of the order (logit descending, index
// ascending), so the kept set is one cut (key, index) in that order plus a bound
// on the exponent, and nothing is sorted. A cut is found by a histogram over
// 2048 bins of (max - l) / T, then, inside the one bin that it falls in, by the
// exact order of the bin's few elements (or by further histograms over the bits
// of their keys, when there are many). The token comes from a walk over running
// masses in index order.
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
constexpr int kCand = 256;     // elements of a bin resolved by their exact order
constexpr int kMaxCluster = 16;
constexpr float kSpan = 32.0f;  // exponents below -kSpan have mass 0: e^-32 < 2^-46

struct SampleParams {
  const void* x;
  int64_t ld;
  int type, V, chunk, S;
  const float *u, *temp, *top_p, *min_p;
  const int32_t* top_k;
  int32_t *tok, *tok2;
  float* logprob;
};

// Order-preserving key of a logit: larger key, larger logit; -0 as +0, NaN as -inf.
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
  uint32_t cnt[kBins];
  uint32_t mass[3][kBins];  // 16-bit limbs of the bins' masses (a CTA holds at most 2^16 elements)
  uint64_t slot[2][kMaxCluster][2];  // values that the CTAs send one another, in turn
  uint64_t warp[kWarps][2];
  uint64_t found[2];      // what this CTA found for the others to read
  uint64_t result[4];
  uint32_t ckey[kCand], cidx[kCand];
  uint64_t cmass[kCand];
  uint32_t ncand;
};

// One row's state, the same in every thread of the cluster.
struct Row {
  uint32_t top;     // key of the largest logit
  float top_value;
  double m, inv_t;  // the largest logit and 1 / T
  float bin_scale;
  double min_e;     // min-p: exponents below are dropped
  int S;
  uint32_t cut_key, cut_idx;  // kept: key > cut_key, or == and idx <= cut_idx
  __device__ __forceinline__ double exponent(uint32_t key) const {
    return key == top ? 0.0 : ((double)key_value(key) - m) * inv_t;  // NaN for -inf at an infinite T
  }
  __device__ __forceinline__ bool alive(uint32_t key) const { return exponent(key) > -(double)kSpan; }
  __device__ __forceinline__ uint64_t weight_of(double e) const { return (uint64_t)rint(exp(e) * (double)(1ull << S)); }
  __device__ __forceinline__ uint64_t weight(uint32_t key) const {
    const double e = exponent(key);
    return e > -(double)kSpan ? weight_of(e) : 0ull;
  }
  // Bin of an element that is alive: fp32 subtraction and product are monotone, so bins follow the order.
  __device__ __forceinline__ int bin(uint32_t key) const {
    if (key == top) return 0;
    return min(kBins - 1, (int)((top_value - key_value(key)) * bin_scale));
  }
  __device__ __forceinline__ bool inside(uint32_t key, uint32_t idx) const {
    return key > cut_key || (key == cut_key && idx <= cut_idx);
  }
};

struct Cluster {
  Shared& sh;
  int rank, size, turn;
  __device__ __forceinline__ uint32_t at(const void* p, int r) const { return mapa_shared(smem_u32(p), r); }
  // Every CTA sends (a, b) (its thread 0's) to all; on return slots() holds all of them. All threads call.
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

// Block sum of two values; every thread gets the totals.
__device__ __forceinline__ void block_sum2(Shared& sh, uint64_t& a, uint64_t& b) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh.warp[threadIdx.x >> 5][0] = a, sh.warp[threadIdx.x >> 5][1] = b;
  __syncthreads();
  a = b = 0;
  for (int i = 0; i < kWarps; ++i) a += sh.warp[i][0], b += sh.warp[i][1];
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

// The bins' values: counts, or masses from their limbs, summed over the cluster.
template <bool MASS>
__device__ __forceinline__ uint64_t bin_value(const Cluster& c, int b) {
  uint64_t v = 0;
  for (int r = 0; r < c.size; ++r) {
    if (MASS)
      v += (uint64_t)ld_cluster_u32(c.at(&c.sh.mass[0][b], r)) + ((uint64_t)ld_cluster_u32(c.at(&c.sh.mass[1][b], r)) << 16) +
           ((uint64_t)ld_cluster_u32(c.at(&c.sh.mass[2][b], r)) << 32);
    else
      v += ld_cluster_u32(c.at(&c.sh.cnt[b], r));
  }
  return v;
}

// The cut of the shortest prefix whose value (count, or mass) reaches a goal.
// GOAL(total) gives the goal from the value of everything inside the present cut
// and returns 0 to leave the cut alone. All threads of the cluster call it, and
// every branch below is the same for all of them.
template <bool MASS, typename Goal>
__device__ void select(Cluster& c, Row& row, const uint32_t* keys, int n, uint32_t idx0, Goal goal_of) {
  Shared& sh = c.sh;
  const int tid = threadIdx.x, per = kBins / c.size, each = (per + kThreads - 1) / kThreads;
  uint64_t before = 0, goal = 0;  // the value of what lies above the range; the goal
  uint32_t lo = 0, hi = 0xffffffffu;  // keys of the range, inclusive
  int shift = 0;
  bool first = true;                  // the first histogram is over the bins of Row::bin
  // bin of an element of the range, or -1
  auto bin_of = [&](uint32_t key, uint32_t idx) -> int {
    if (!row.inside(key, idx) || !row.alive(key)) return -1;
    if (first) return row.bin(key);
    if (key < lo || key > hi) return -1;
    return (int)((hi - key) >> shift);
  };
  for (int pass = 0; pass < 6; ++pass) {  // at most 4 are needed: 2048 bins, then 11 bits of the key each
    __syncthreads();
    for (int b = tid; b < kBins; b += kThreads) {
      sh.cnt[b] = 0;
      if (MASS) sh.mass[0][b] = sh.mass[1][b] = sh.mass[2][b] = 0;
    }
    if (tid == 0) sh.ncand = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kThreads) {
      const int b = bin_of(keys[i], idx0 + i);
      if (b < 0) continue;
      atomicAdd(&sh.cnt[b], 1u);
      if (MASS) {
        const uint64_t w = row.weight(keys[i]);
        atomicAdd(&sh.mass[0][b], (uint32_t)(w & 0xffffu));
        atomicAdd(&sh.mass[1][b], (uint32_t)((w >> 16) & 0xffffu));
        atomicAdd(&sh.mass[2][b], (uint32_t)(w >> 32));
      }
    }
    __syncthreads();
    cluster_barrier();
    // this CTA's slice of the bins, each thread `each` bins in order
    uint64_t mine = 0;
    const int s0 = c.rank * per;
    for (int e = 0; e < each; ++e) {
      const int b = tid * each + e;
      if (b < per) mine += bin_value<MASS>(c, s0 + b);
    }
    uint64_t slice;
    const uint64_t pre = block_scan(sh, mine, &slice);
    const auto slots = c.exchange(slice, 0);
    uint64_t total = 0, above = before;
    for (int r = 0; r < c.size; ++r) {
      if (r < c.rank) above += slots[r][0];
      total += slots[r][0];
    }
    if (first) {
      goal = goal_of(total);
      if (goal == 0) return;  // (the same in every thread of the cluster)
    }
    // the thread whose bins the goal falls in finds the bin
    if (tid == 0) sh.found[0] = ~0ull;
    __syncthreads();
    uint64_t run = above + pre;
    if (run < goal && goal <= run + mine) {
      for (int e = 0; e < each; ++e) {
        const int b = s0 + tid * each + e;
        const uint64_t v = bin_value<MASS>(c, b);
        if (run < goal && goal <= run + v) {
          sh.found[0] = ((uint64_t)b << 32) | (uint32_t)bin_value<false>(c, b);
          sh.found[1] = run;
        }
        run += v;
      }
    }
    __syncthreads();
    const auto got = c.exchange(sh.found[0], sh.found[1]);
    int bin = 0;
    uint32_t count = 0;
    for (int r = 0; r < c.size; ++r)
      if (got[r][0] != ~0ull) {
        bin = (int)(got[r][0] >> 32);
        count = (uint32_t)got[r][0];
        before = got[r][1];
      }
    const bool single = !first && shift == 0;  // every element of the bin has the same key
    if (count <= (uint32_t)kCand) {
      // the bin's elements to CTA 0, which puts them in their exact order
      for (int i = tid; i < n; i += kThreads) {
        if (bin_of(keys[i], idx0 + i) != bin) continue;
        const uint32_t at = atom_cluster_inc(c.at(&sh.ncand, 0));
        if (at >= (uint32_t)kCand) continue;
        st_cluster_b32(c.at(&sh.ckey[at], 0), keys[i]);
        st_cluster_b32(c.at(&sh.cidx[at], 0), idx0 + i);
      }
      cluster_barrier();
      if (c.rank == 0) {
        const int m = (int)min(count, (uint32_t)kCand);
        for (int i = tid; i < m; i += kThreads) sh.cmass[i] = MASS ? row.weight(sh.ckey[i]) : 1ull;
        if (tid == 0) sh.found[0] = sh.found[1] = 0;
        __syncthreads();
        // two threads per element: the value of what precedes it in the bin
        const int i = tid >> 1;
        uint64_t v = 0;
        if (i < m) {
          const uint32_t ki = sh.ckey[i], xi = sh.cidx[i];
          for (int j = tid & 1; j < m; j += 2) {
            const uint32_t kj = sh.ckey[j];
            if (kj > ki || (kj == ki && sh.cidx[j] < xi)) v += sh.cmass[j];
          }
        }
        v += __shfl_xor_sync(0xffffffffu, v, 1);
        if (i < m && (tid & 1) == 0 && before + v < goal && goal <= before + v + sh.cmass[i]) {
          sh.found[0] = sh.ckey[i];
          sh.found[1] = sh.cidx[i];
        }
        __syncthreads();
      }
      const auto cut = c.exchange(sh.found[0], sh.found[1]);
      row.cut_key = (uint32_t)cut[0][0];
      row.cut_idx = (uint32_t)cut[0][1];
      return;
    }
    if (single) {
      // many equal keys: the goal's place among them, in index order
      const uint32_t key = hi - bin;
      const uint64_t g = MASS ? row.weight(key) : 1ull;
      const uint64_t need = (goal - before + g - 1) / g;  // ties to keep, >= 1
      uint64_t ties = 0, unused = 0;
      const int blk = (n + kThreads - 1) / kThreads, i0 = min(n, tid * blk), i1 = min(n, i0 + blk);
      for (int i = i0; i < i1; ++i) ties += keys[i] == key && row.inside(key, idx0 + i);
      uint64_t all;
      const uint64_t tpre = block_scan(sh, ties, &all);
      const auto tslots = c.exchange(all, unused);
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
      return;
    }
    if (first) {
      // the bin's keys: their least and greatest bound the next histogram
      uint32_t kmin = 0xffffffffu, kmax = 0;
      for (int i = tid; i < n; i += kThreads)
        if (bin_of(keys[i], idx0 + i) == bin) kmin = min(kmin, keys[i]), kmax = max(kmax, keys[i]);
      kmin = __reduce_min_sync(0xffffffffu, kmin);
      kmax = __reduce_max_sync(0xffffffffu, kmax);
      __syncthreads();
      if ((tid & 31) == 0) sh.warp[tid >> 5][0] = kmin, sh.warp[tid >> 5][1] = kmax;
      __syncthreads();
      for (int i = 0; i < kWarps; ++i) kmin = min(kmin, (uint32_t)sh.warp[i][0]), kmax = max(kmax, (uint32_t)sh.warp[i][1]);
      const auto ks = c.exchange(kmin, kmax);
      for (int r = 0; r < c.size; ++r) kmin = min(kmin, (uint32_t)ks[r][0]), kmax = max(kmax, (uint32_t)ks[r][1]);
      lo = kmin;
      hi = kmax;
      first = false;
    } else {
      const uint32_t top = hi - ((uint32_t)bin << shift), width = (1u << shift) - 1;
      hi = top;
      lo = top - lo > width ? top - width : lo;
    }
    const int bits = hi > lo ? 32 - __clz(hi - lo) : 0;  // hi - lo < 2^bits
    shift = max(0, bits - 11);
  }
}

__global__ void __launch_bounds__(kThreads) sample_kernel(const __grid_constant__ SampleParams p) {
  extern __shared__ uint32_t keys[];
  __shared__ Shared sh;
  uint32_t size, rank;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(size));
  rank = cluster_ctarank();
  Cluster c{sh, (int)rank, (int)size, 0};
  pdl_launch_dependents();
  pdl_wait();
  const int b = blockIdx.x / size, tid = threadIdx.x;
  const int idx0 = min(p.V, (int)rank * p.chunk), n = min(p.V - idx0, p.chunk);
  // the chunk's keys, and its largest with the lowest index
  uint64_t best = 0;
  {
    const int64_t o = (int64_t)b * p.ld + idx0;
    auto put = [&](int i, float v) {
      const uint32_t k = key_of(v);
      keys[i] = k;
      const uint64_t cand = ((uint64_t)k << 32) | (uint32_t)~(idx0 + i);
      best = cand > best ? cand : best;
    };
    if (p.type == BTF_F32) {
      const float* x = static_cast<const float*>(p.x) + o;
      for (int i = tid; i < n; i += kThreads) put(i, x[i]);
    } else if (p.type == BTF_F16) {
      const __half* x = static_cast<const __half*>(p.x) + o;
      for (int i = tid; i < n; i += kThreads) put(i, __half2float(x[i]));
    } else {
      const __nv_bfloat16* x = static_cast<const __nv_bfloat16*>(p.x) + o;
      for (int i = tid; i < n; i += kThreads) put(i, __bfloat162float(x[i]));
    }
  }
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
  const float T = p.temp ? p.temp[b] : 1.0f;
  const bool none = row.top <= kNegInf;
  if (none || !(T > 0.0f)) {  // nothing to draw from, or greedy
    cluster_barrier();        // no CTA leaves while another may still write its slots
    if (rank == 0 && tid == 0) {
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
  {
    const float mp = p.min_p ? p.min_p[b] : 0.0f;
    row.min_e = mp > 0.0f ? fmin(log((double)mp), 0.0) : -INFINITY;
  }
  const int k = p.top_k ? p.top_k[b] : 0;
  if (k > 0 && k < p.V)
    select<false>(c, row, keys, n, idx0, [k](uint64_t total) { return (uint64_t)k < total ? (uint64_t)k : 0ull; });
  const float tp = p.top_p ? p.top_p[b] : 1.0f;
  if (tp < 1.0f)
    select<true>(c, row, keys, n, idx0, [tp](uint64_t total) {
      const double g = ceil((double)tp * (double)total);
      return g < 1.0 ? 1ull : (uint64_t)g < total ? (uint64_t)g : total;
    });
  // running masses in index order: a warp owns a contiguous block
  const int lane = tid & 31, w = tid >> 5, blk = (n + kWarps - 1) / kWarps;
  const int w0 = min(n, w * blk), w1 = min(n, w0 + blk);
  auto kept = [&](int i) -> uint64_t {
    const uint32_t key = keys[i];
    if (!row.inside(key, idx0 + i)) return 0ull;
    const double e = row.exponent(key);
    return e > -(double)kSpan && e >= row.min_e ? row.weight_of(e) : 0ull;
  };
  uint64_t mine = 0;
  for (int i = w0 + lane; i < w1; i += 32) mine += kept(i);
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
  const double u = (double)p.u[b];
  const double goal_d = u > 0.0 ? u * (double)z : 0.0;
  const uint64_t goal = goal_d < (double)z ? min((uint64_t)goal_d, z - 1) : z - 1;
  if (pre <= goal && goal < pre + mine) {
    // the warp that holds the token walks its block
    uint64_t run = pre;
    for (int i0 = w0; i0 < w1; i0 += 32) {
      const uint64_t v = i0 + lane < w1 ? kept(i0 + lane) : 0ull;
      uint64_t inc = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint64_t q = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += q;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, run + inc > goal);
      if (hit) {
        if (lane == __ffs(hit) - 1) {
          const int32_t t = idx0 + i0 + lane;
          p.tok[b] = t;
          if (p.tok2) p.tok2[b] = t;
          if (p.logprob)
            p.logprob[b] = (float)(row.exponent(keys[i0 + lane]) - log((double)z / (double)(1ull << row.S)));
        }
        break;
      }
      run += __shfl_sync(0xffffffffu, inc, 31);
    }
  }
}

}  // namespace

int sample_setup(DeviceInfo& d) {
  constexpr int kMost = BTF_SAMPLE_MAX_V / kMaxCluster * 4;  // the largest chunk's keys
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
  p.chunk = (a.V + size - 1) / size;
  return launch_pdl_cluster(sample_kernel, dim3((unsigned)(a.B * size)), dim3(kThreads), (size_t)p.chunk * 4, st, size,
                            p);
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
