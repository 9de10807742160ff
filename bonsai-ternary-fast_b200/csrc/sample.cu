// Sampling from given random numbers (btf_sample): temperature, top-k, top-p and
// min-p on one row of logits per thread-block cluster. With few rows a CTA keeps its
// part of the row in shared memory; with many (more CTAs than are resident at once)
// fewer CTAs a row keep a summary of it (the largest of every 16 logits of a lane)
// and read again only what a pass needs.
//
// All three filters keep a prefix of the order (logit descending, index
// ascending), so nothing is sorted: a cut (key, index) in that order plus a bound on
// the exponent is the kept set. What bounds the kernel is the number of passes over
// the row and of exchanges through the cluster (1 to 1.8 us each with what is sent,
// 0.24 of it the bare barrier), so the common cases take few:
//   top-k: a histogram of each thread's largest logit (of its 32 or so) gives a bound
//     that at least k logits reach and few more than k exceed; those go to the
//     cluster's first CTA, which ranks them exactly and finishes the row: 3 barriers;
//   top-p: a histogram of counts over 8192 bins of (max - l) / T, times the bins'
//     middle masses, points at a few bins with the cut among them. The exact mass
//     above them and their elements, ranked by the first CTA, give the cut or show that
//     it lies elsewhere (then exact histograms find it). Few elements down to there:
//     the first CTA finishes the row. Else the token comes from a walk over running
//     masses in index order, each CTA over its own part of the row;
//   no such filter: the walk alone: 2 barriers.
// The walk sums up every warp's block of the row; the one block with the token is then
// shared out among the CTA's warps, and one of them goes through its share.
// Bounds on (max - l) / T are turned into bounds on keys once, so that a pass over the
// row compares integers and only what it keeps is worked out.
//
// Masses are 64-bit integers, w = rint(exp((l - max) / T) 2^S): sums are exact in
// any order, so the CTAs of a cluster, the histogram and the final walk agree on
// every total to the last bit, and the drawn token is a function of the inputs
// alone. S = 62 - ceil(log2 V) (44 for V up to 2^18): a mass is off by 2^-45 of
// the largest one; exponents are taken in 64 bits, since a token next to a border
// of the running mass would go the other way under the 2^-24 of fp32.
//
// Measured (device time, the logits not in L2): 1 row of 248320 fp32, top-k 50 and
// top-p 0.95: 13.9 us, in which no phase stands out (cold, by cycle counts of one CTA,
// 15.2 us: start 0.7, reading 2.3, three exchanges 4.3, the histogram 0.6, the searches
// for the bin and its bounds 2.4, the ranking 1.9, masses 0.8, index order 1.2, the draw 1.0);
// 7 x 128003, top-p 0.9: 27.1 (three passes over what shared memory holds, two lists
// ranked); 33 x 50257 bf16, top-k, top-p and min-p: 18.5; 64 x 248320, min-p: 24.8,
// 63.6 MB at 2.6 TB/s, the reading at 6.3. Without a filter 64 x 248320 take 57: the
// 64-bit exponents of all 16 M logits bound it.
#include <algorithm>
#include <cmath>

#include "elem.cuh"
#include "sample.h"

namespace btf {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 2048;    // of exact histograms
constexpr int kFine = 8192;    // of counts
constexpr int kGroups = 64;    // of bins, summed for the whole cluster's use
constexpr int kCand = 512;     // elements that one CTA ranks exactly, one per thread
constexpr int kMaxCluster = 16;
constexpr int kHeld = 16384;   // logits that a CTA keeps in shared memory at most
constexpr int kLeast = 4096;   // and at least, while there are SMs without a CTA
constexpr float kSpan = 32.0f;  // exponents below -kSpan have mass 0: e^-32 < 2^-46

struct SampleParams {
  const void* x;
  int64_t ld;
  int V, chunk, S;  // chunk: logits per CTA, a multiple of 4 x kThreads
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
__device__ __forceinline__ uint4 ld_cluster_v4(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(a)
               : "memory");
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
  uint64_t group[kMaxCluster][kGroups];  // every CTA's sums of the groups of its bins
  float square[kMaxCluster][kGroups];    // and of the squares of their elements' masses, in 2^S
  uint64_t total[kMaxCluster], above[kMaxCluster];  // every CTA's masses
  uint64_t end[2];
  int end_bin[2];
  uint64_t warp[kWarps][2];
  uint64_t found[2];
  int found_bin;
  double exp2_64[64];  // 2^(i / 64)
  uint64_t cmass[kCand];
  uint32_t ckey[kCand], cidx[kCand];
  uint32_t ncand;
};
// A histogram of counts, or an exact one of counts or masses.
union Hist {
  uint32_t cnt[kFine];
  unsigned long long bin[kBins];
};
struct Queue {  // logits whose masses a warp works out, 32 at a time (in the histogram's place: that is done by then)
  float of[kWarps][32 + 4 * 32];
};
static_assert(sizeof(Queue) <= sizeof(Hist));

// One row's state, the same in every thread of the cluster.
struct Row {
  float top;        // the largest logit
  double m, inv_t;  // it and 1 / T
  float bin_scale;
  double min_e;     // min-p: exponents below are dropped
  float alive;      // logits below have no mass
  int S;
  float cut;        // kept: above the cut, or equal to it and idx <= cut_idx
  uint32_t cut_idx;
  const double* table;

  __device__ __forceinline__ double exponent(float v) const { return v == top ? 0.0 : ((double)v - m) * inv_t; }
  // (max - l) / T in bins: fp32 subtraction and product are monotone, so it follows the order. At least kBins, or
  // NaN, has no mass.
  __device__ __forceinline__ float place(float v) const { return v == top ? 0.0f : (top - v) * bin_scale; }
  // rint(2^S e^x) for -33 < x <= 0 by a table of 2^(i / 64) and the Taylor polynomial of the rest (Tang's method):
  // x = n ln2 / 64 + r, |r| <= ln2 / 128, e^r to r^5 / 120 (the rest below 2^-54), in all within 2^-48 relative. (16
  // entries, whose lookups do not conflict, and one term more: the same time.)
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
  __device__ __forceinline__ uint64_t weight(float v) const { return v >= alive ? weight_of(exponent(v)) : 0ull; }
  // The least number above -inf with a place below `bound` > 0, for a converged warp: around where it should be,
  // then by a 32-way search over the keys.
  __device__ __forceinline__ float least(float bound) const {
    const uint32_t end = key_of(top);
    uint32_t lo = kNegInf, hi = end;  // lo fails, hi holds
    const int lane = threadIdx.x & 31;
    auto narrow = [&](uint32_t k) {
      const bool holds = place(key_value(k)) < bound;
      hi = min(hi, __reduce_min_sync(0xffffffffu, holds ? k : end));
      lo = max(lo, __reduce_max_sync(0xffffffffu, holds ? kNegInf : k));
    };
    const float at = top - bound / bin_scale;
    if (hi - lo > 32 && fabsf(at) < INFINITY) {
      const uint32_t g = key_of(at), d = 1u << (2 * (lane & 15));
      const uint32_t k = lane < 16 ? (g > kNegInf + d ? g - d : kNegInf + 1) : (end - kNegInf > d && g < end - d ? g + d : end);
      narrow(min(max(k, kNegInf + 1), end));
    }
    while (hi - lo > 1) narrow(lo + 1 + (uint32_t)(((uint64_t)(hi - lo - 1) * lane) >> 5));
    return key_value(hi);
  }
  __device__ __forceinline__ bool inside(float v, uint32_t idx) const { return v > cut || (v == cut && idx <= cut_idx); }
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

// A CTA's part of the row, in fours of neighbours as fp32: in shared memory (HELD), or where it lies. A warp owns a
// contiguous block of `blk` fours, its lanes one after another. What pads the last four is -inf.
constexpr int kGroup = 4;
constexpr int kHits = 256;  // of a warp's groups, 8 rounds of 32, that are listed at a time
template <typename T, bool HELD>
struct Part {
  float4* held;
  __nv_bfloat16* peak;  // or the largest of every lane's kGroup fours, rounded up,
  uint16_t* hits;       // and this warp's list of those that a pass has to read
  const T* x;
  int n, blk;     // logits; fours per warp
  bool whole;     // whether fours are aligned
  float largest;  // of this thread's
  __device__ __forceinline__ float4 raw(int i) const {
    float v[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    const int left = n - 4 * i;
    if (whole && left >= 4) {
      Pack<T, 4> w;
      w.load(x + 4 * (int64_t)i);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = w.get(e);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < left) v[e] = to_f32(x[4 * (int64_t)i + e]);
    }
    return make_float4(v[0], v[1], v[2], v[3]);
  }
  __device__ __forceinline__ float4 four(int i) const {
    if constexpr (HELD) return held[i];
    else return raw(i);
  }
  // fn(four, position in the part) with the whole warp, for the fours of which a lane's holds a logit >= from
  template <typename Fn>
  __device__ __forceinline__ void fours(float from, Fn fn) const {
    const bool none = !(largest >= from);
    if (__all_sync(0xffffffffu, none)) return;
    const int i0 = (threadIdx.x >> 5) * blk, i1 = i0 + blk, lane = threadIdx.x & 31;
    const float4 nothing = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    // this lane's fours i, i + 32, ...; one copy of fn for all of them: the code stays small
    constexpr int kAhead = 2;
    static_assert(kGroup % kAhead == 0);
    auto some = [&](int i, bool any) {
      float4 q[kAhead];
#pragma unroll
      for (int a = 0; a < kAhead; ++a) q[a] = any && i + 32 * a < i1 ? four(i + 32 * a) : nothing;
#pragma unroll 1
      for (int a = 0; a < kAhead; ++a) {
        const float4 f = q[0];
#pragma unroll
        for (int b = 0; b + 1 < kAhead; ++b) q[b] = q[b + 1];
        if (__any_sync(0xffffffffu, fmaxf(fmaxf(f.x, f.y), fmaxf(f.z, f.w)) >= from)) fn(f, 4 * (i + 32 * a));
      }
    };
    if constexpr (HELD) {
#pragma unroll 1
      for (int i = i0 + lane; i < i1; i += 32 * kAhead) some(i, !none);
    } else {
      // the groups with something to read are listed and read a lane each: few of them take one trip to memory
      const int groups = (blk + 32 * kGroup - 1) / (32 * kGroup);
#pragma unroll 1
      for (int g0 = 0; g0 < groups; g0 += kHits / 32) {
        int n = 0;
#pragma unroll 1
        for (int g = g0; g < min(g0 + kHits / 32, groups); ++g) {
          const bool is = __bfloat162float(peak[g * 32 + lane]) >= from;
          const unsigned are = __ballot_sync(0xffffffffu, is);
          if (is) hits[n + __popc(are & ((1u << lane) - 1))] = (uint16_t)(g * 32 + lane);
          n += __popc(are);
        }
        __syncwarp();
#pragma unroll 1
        for (int h = lane; h < n + lane; h += 32) {
          const int e = h < n ? hits[h] : 0;
#pragma unroll 1
          for (int a = 0; a < kGroup; a += kAhead) some(i0 + e / 32 * (32 * kGroup) + e % 32 + 32 * a, h < n);
        }
        __syncwarp();
      }
    }
  }
  // fn(logit, position in the part) for this thread's fours that hold a logit >= from
  template <typename Fn>
  __device__ __forceinline__ void each(float from, Fn fn) const {
    fours(from, [&](const float4& f, int at) {
      if (!(fmaxf(fmaxf(f.x, f.y), fmaxf(f.z, f.w)) >= from)) return;
      fn(f.x, at);
      fn(f.y, at + 1);
      fn(f.z, at + 2);
      fn(f.w, at + 3);
    });
  }
};

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
  if (threadIdx.x < kGroups)
    for (int r = 0; r < c.size; ++r) v += c.sh.group[r][threadIdx.x];
  return block_sum(c.sh, v);
}

// The bin in which the running value (from the largest logits on, `before` ahead of the first) reaches the goal,
// over the whole cluster's histograms: every CTA finds it for itself.
struct Found {
  int bin;
  uint64_t before, value, all;  // all: of the whole histogram; less than the goal: the rest means nothing
};
__device__ __forceinline__ Found find_bin(const Cluster& c, uint64_t before, uint64_t goal) {
  Shared& sh = c.sh;
  uint64_t v = 0, all;
  if (threadIdx.x < kGroups)
    for (int r = 0; r < c.size; ++r) v += sh.group[r][threadIdx.x];
  const uint64_t run = before + block_scan(sh, v, &all);
  if (run < goal && goal <= run + v) {
    sh.found[0] = run;
    sh.found_bin = threadIdx.x;
  }
  __syncthreads();
  if (before + all >= goal && threadIdx.x < 32) {  // the group's bins, a lane each
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
  const Found f{sh.found_bin, sh.found[0], sh.found[1], all};
  __syncthreads();
  return f;
}

__device__ __forceinline__ uint64_t goal_of_u(float uf, uint64_t z) {
  const double u = (double)uf, g = u > 0.0 ? u * (double)z : 0.0;
  return g < (double)z ? min((uint64_t)g, z - 1) : z - 1;
}
__device__ __forceinline__ void put_token(const SampleParams& p, int b, const Row& row, float v, uint32_t idx,
                                          uint64_t z) {
  p.tok[b] = (int32_t)idx;
  if (p.tok2) p.tok2[b] = (int32_t)idx;
  if (p.logprob) p.logprob[b] = (float)(row.exponent(v) - log((double)z / (double)(1ull << row.S)));
}

// The share of `total` that top-p keeps, rounded up: the prefix ends with the element that reaches it.
__device__ __forceinline__ uint64_t goal_of_p(float p, uint64_t total) {
  const double g = ceil((double)p * (double)total);
  return g < 1.0 ? 1ull : (uint64_t)g < total ? (uint64_t)g : total;
}

// Bitonic sort of one value per thread, the largest first; those of the threads from n on are 0. `buf` holds
// kThreads values.
template <typename U>
__device__ __forceinline__ U sorted(U v, int n, U* buf) {
  const int tid = threadIdx.x;
#pragma unroll 1
  for (int k = 2; k < 2 * n; k <<= 1) {
#pragma unroll 1
    for (int j = k >> 1; j > 0; j >>= 1) {
      U o;
      if (j >= 32) {
        __syncthreads();
        buf[tid] = v;
        __syncthreads();
        o = buf[tid ^ j];
      } else {
        o = __shfl_xor_sync(0xffffffffu, v, j);
      }
      v = (((tid & j) == 0) == ((tid & k) == 0)) == (v > o) ? v : o;
    }
  }
  __syncthreads();
  return v;
}
// The first CTA's list in the row's order, one per thread (0: none): key above, ~index below.
__device__ __forceinline__ uint64_t sorted_list(Shared& sh) {
  const int tid = threadIdx.x, n = (int)min(sh.ncand, (uint32_t)kCand);
  return sorted<uint64_t>(tid < n ? ((uint64_t)sh.ckey[tid] << 32) | (uint32_t)~sh.cidx[tid] : 0ull, n, sh.cmass);
}

// The cluster's first CTA finishes a row from its list of candidates, which holds
// every element down to the cut. k: elements to keep; goal: mass to reach, or with
// RANKED top_p of the first k's.
template <bool RANKED>
__device__ void finish(Shared& sh, const SampleParams& p, int b, const Row& row, uint64_t k, uint64_t goal, float top_p) {
  const int tid = threadIdx.x, n = (int)min(sh.ncand, (uint32_t)kCand);
  const uint64_t v = sorted_list(sh);
  const uint32_t key = (uint32_t)(v >> 32), idx = ~(uint32_t)v;
  const float logit = key_value(key);
  const uint64_t w = v ? row.weight(logit) : 0;
  uint64_t all;
  const uint64_t before = block_scan(sh, w, &all);
  bool keep = w > 0;
  if (RANKED) {
    keep = keep && (uint64_t)tid < k;
    const uint64_t zk = block_sum(sh, keep ? w : 0);
    goal = top_p < 1.0f ? goal_of_p(top_p, zk) : zk;
  }
  keep = keep && before < goal && row.exponent(logit) >= row.min_e;
  // the running mass in index order: (index, rank) sorted, the least index last
  static_assert(BTF_SAMPLE_MAX_V <= (1 << 19) && kCand == 1 << 9);
  __syncthreads();
  const uint32_t s = sorted<uint32_t>(keep ? ((idx + 1) << 9) | tid : 0u, n, reinterpret_cast<uint32_t*>(sh.cmass));
  sh.cmass[tid] = keep ? w : 0;
  sh.ckey[tid] = key;
  __syncthreads();
  const uint64_t mass = s ? sh.cmass[s & (kCand - 1)] : 0;
  uint64_t z;
  const uint64_t down = block_scan(sh, mass, &z);  // the mass of the indices behind this one
  const uint64_t g = goal_of_u(p.u[b], z);
  const uint64_t run = z - down - mass;            // and of those before it
  if (mass && run <= g && g < run + mass) put_token(p, b, row, key_value(sh.ckey[s & (kCand - 1)]), (s >> 9) - 1, z);
}

// Sends this CTA's logits from lo on and not from `end` on (NaN: no end), inside the cut, to the first CTA's list;
// fn(logit, position) for every one from lo on.
template <typename P, typename Fn>
__device__ __forceinline__ void collect(const Cluster& c, const Row& row, const P& part, uint32_t idx0, float lo,
                                        float end, Fn fn) {
  const uint32_t n_at = c.at(&c.sh.ncand, 0), key_at = c.at(c.sh.ckey, 0), idx_at = c.at(c.sh.cidx, 0);
  part.each(lo, [&](float v, int i) {
    if (!(v >= lo) || !row.inside(v, idx0 + i)) return;
    fn(v, i);
    if (v >= end) return;
    const uint32_t at = atom_cluster_inc(n_at);
    if (at >= (uint32_t)kCand) return;
    st_cluster_b32(key_at + at * 4, key_of(v));
    st_cluster_b32(idx_at + at * 4, idx0 + i);
  });
}
// The barrier after it; how many there were in all: at most kCand of them are in the list.
__device__ __forceinline__ uint32_t collected(const Cluster& c) {
  cluster_barrier();
  return ld_cluster_u32(c.at(&c.sh.ncand, 0));
}

// The first CTA ranks its list and sends the cut to all: the element that carries the value from `before` to the
// goal. False if there is none.
template <bool MASS>
__device__ __forceinline__ bool cut_of_list(Cluster& c, Row& row, uint64_t before, uint64_t goal) {
  Shared& sh = c.sh;
  const int tid = threadIdx.x;
  if (c.rank == 0) {
    const uint64_t v = sorted_list(sh);
    const uint64_t w = v ? MASS ? row.weight(key_value((uint32_t)(v >> 32))) : 1ull : 0ull;
    if (tid == 0) sh.found[0] = 0;
    uint64_t all;
    const uint64_t run = before + block_scan(sh, w, &all);  // (its barriers are between the two writes)
    if (run < goal && goal <= run + w) {
      sh.found[0] = v >> 32;  // (no logit has key 0)
      sh.found[1] = (uint32_t)~(uint32_t)v;
    }
    __syncthreads();
  }
  const auto cut = c.exchange(sh.found[0], sh.found[1]);
  if (cut[0][0] == 0) return false;
  row.cut = key_value((uint32_t)cut[0][0]);
  row.cut_idx = (uint32_t)cut[0][1];
  return true;
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

__device__ __forceinline__ float no_end() { return __uint_as_float(0x7fc00000u); }

// Top-k from the threads' largest logits (see the top): true when the row is
// finished, false when there are too few or too many for it. All threads of the
// cluster call it.
template <typename P>
__device__ bool top_of_threads(Cluster& c, const SampleParams& p, int b, Row& row, const P& part, uint32_t idx0,
                               uint64_t k, float top_p) {
  if (part.largest >= row.alive) atomicAdd(&c.hist.bin[(int)row.place(part.largest)], 1ull);
  if (threadIdx.x == 0) c.sh.ncand = 0;
  publish(c);
  bool done = false;
  const Found f = find_bin(c, 0, k);
  if (f.all >= k && f.before + f.value <= (uint64_t)kCand) {
    collect(c, row, part, idx0, row.least((float)(f.bin + 1)), no_end(), [](float, int) {});
    done = collected(c) <= (uint32_t)kCand;
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

// The cut by a histogram of counts (see the top). kFailed: it takes exact
// histograms; the present one is clear then, as on entry. kCut: `above` is this
// warp's mass of the logits from `upto` on. All threads of the cluster call it.
enum Outcome { kFailed, kCut, kFinished };
template <bool MASS, typename P>
__device__ Outcome cut_by_counts(Cluster& c, const SampleParams& p, int row_b, Row& row, const P& part, uint32_t idx0,
                                 uint64_t k, float top_p, uint64_t* above, float* upto) {
  Shared& sh = c.sh;
  const int tid = threadIdx.x, lane = tid & 31;
  constexpr float kPer = kFine / kBins;  // fine bins per bin of Row::place
  constexpr double kWidth = (double)kSpan / kFine;
  // the middle mass of a fine bin, within 2^-20
  const float one = (float)(1ull << row.S);
  auto middle = [&](int bin) { return exp2f((bin + 0.5f) * (float)(-kWidth * 1.4426950408889634)) * one; };
  uint64_t sum = 0;
  part.each(row.alive, [&](float v, int i) {
    if (!(v >= row.alive) || !row.inside(v, idx0 + i)) return;
    atomicAdd(&c.hist.cnt[(int)(row.place(v) * kPer)], 1u);
    sum += MASS ? row.weight_of(row.exponent(v)) : 1ull;
  });
  sum = block_sum(sh, sum);
  if (tid < c.size) st_cluster_u64(c.at(&sh.total[c.rank], tid), sum);
  if (tid == 0) sh.ncand = 0;
  constexpr int kOf = kFine / kGroups;  // bins of a group: 4 per lane
  static_assert(kOf == 128);
  for (int g = tid >> 5; g < kGroups; g += kWarps) {
    const int b0 = g * kOf + lane * 4;
    const uint4 q = *reinterpret_cast<const uint4*>(&c.hist.cnt[b0]);
    uint64_t v = (uint64_t)q.x + q.y + q.z + q.w;
    float v2 = 0.f;
    if (MASS) {
      float v1 = 0.f;
      if (v) {
        const float mid = middle(b0), f = mid / one;
        v1 = mid * (float)q.x + middle(b0 + 1) * (float)q.y + middle(b0 + 2) * (float)q.z + middle(b0 + 3) * (float)q.w;
        v2 = (float)v * f * f;
      }
      v1 = warp_sum(v1);
      v2 = warp_sum(v2);
      v = (uint64_t)v1;
    } else {
#pragma unroll
      for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    }
    if (lane < c.size) {
      st_cluster_u64(c.at(&sh.group[c.rank][g], lane), v);
      if (MASS) st_cluster_b32(c.at(&sh.square[c.rank][g], lane), __float_as_uint(v2));
    }
  }
  cluster_barrier();
  uint64_t total = 0;
  for (int r = 0; r < c.size; ++r) total += sh.total[r];
  const uint64_t goal = MASS ? goal_of_p(top_p, total) : k;
  if (!MASS && goal >= total) {  // nothing to cut off
    cluster_barrier();           // (the sums are read before they are written again)
    *upto = no_end();
    *above = 0;
    return kCut;
  }
  // the bins of a window around the goal, which the cut is in: an element's mass is off its bin's middle by up to
  // kWidth / 2, evenly spread (kWidth / sqrt 12), so the sums are by that times the root of the sum of squares: four
  // of it, and the rounding of the middles
  uint64_t v = 0, all, slack = 0;
  float v2 = 0.f;
  if (tid < kGroups)
    for (int r = 0; r < c.size; ++r) {
      v += sh.group[r][tid];
      if (MASS) v2 += sh.square[r][tid];
    }
  const uint64_t run = block_scan(sh, v, &all);
  if (MASS) {
    // (of the groups that begin above the goal; the sum of non-negative floats in a fixed order)
    float sq = run < goal ? v2 : 0.f;
    sq = warp_sum(sq);
    if ((tid & 31) == 0) sh.warp[tid >> 5][1] = __float_as_uint(sq);
    __syncthreads();
    sq = 0.f;
    for (int i = 0; i < kGroups / 32; ++i) sq += __uint_as_float((uint32_t)sh.warp[i][1]);
    slack = (uint64_t)(4.0 * kWidth / 3.4641016 * (double)sqrtf(sq) * (double)(1ull << row.S)) + (goal >> 19) + 1;
  }
  const uint64_t ends[2] = {goal > slack ? goal - slack : 1, min(goal + slack, all)};
  const bool reached = goal <= all + slack && ends[0] <= ends[1] && all > 0;
#pragma unroll
  for (int e = 0; e < 2; ++e)
    if (run < ends[e] && ends[e] <= run + v) {
      sh.end[e] = run;
      sh.end_bin[e] = tid;
    }
  __syncthreads();
  if (reached && tid < 64) {  // a warp for either end
    const int which = tid >> 5;
    const uint64_t end = which ? ends[1] : ends[0];
    const int b0 = sh.end_bin[which] * kOf + lane * 4;
    uint4 q = make_uint4(0, 0, 0, 0);
#pragma unroll 4
    for (int r = 0; r < c.size; ++r) {
      const uint4 a = ld_cluster_v4(c.at(&c.hist.cnt[b0], r));
      q.x += a.x, q.y += a.y, q.z += a.z, q.w += a.w;
    }
    uint64_t w[4] = {q.x, q.y, q.z, q.w}, inc = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (MASS) w[e] = (uint64_t)((float)w[e] * middle(b0 + e));
      inc += w[e];
    }
    const uint64_t mine = inc;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t up = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += up;
    }
    uint64_t from = sh.end[which] + inc - mine;
    __syncwarp();
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (from < end && end <= from + w[e]) {
        sh.end[which] = which ? from + w[e] : from;  // the values before the window and down to its end
        sh.end_bin[which] = b0 + e;
      }
      from += w[e];
    }
  }
  __syncthreads();
  const int bin = sh.end_bin[0], last = sh.end_bin[1];
  const uint64_t before = sh.end[0], value = sh.end[1] - before;
  __syncthreads();
  Outcome out = kFailed;
  if (reached) {
    const float lo = row.least((last + 1) / kPer), end = bin ? row.least(bin / kPer) : no_end();
    const uint64_t most = (uint64_t)kCand * (MASS ? row.weight(lo) : 1);
    const bool down = before + value <= most;
    if (down || value <= most) {
      // the exact mass above the window (or down to its end)
      const float over = down ? lo : end;
      uint64_t mass = 0;
      collect(c, row, part, idx0, lo, down ? no_end() : end, [&](float v, int) {
        if (MASS && v >= over) mass += row.weight_of(row.exponent(v));
      });
      if (MASS) {
#pragma unroll
        for (int o = 16; o; o >>= 1) mass += __shfl_xor_sync(0xffffffffu, mass, o);
        *above = mass;
        const uint64_t cta = block_sum(sh, lane == 0 ? mass : 0);
        if (tid < c.size) st_cluster_u64(c.at(&sh.above[c.rank], tid), cta);
      }
      const uint32_t m = collected(c);
      uint64_t exact = before;
      if (MASS) {
        exact = 0;
        for (int r = 0; r < c.size; ++r) exact += sh.above[r];
      }
      if (m <= (uint32_t)kCand) {
        if (down) {
          if (!MASS || goal <= exact) {
            last_read(c, [&] { finish<!MASS>(sh, p, row_b, row, k, goal, top_p); });
            return kFinished;
          }
        } else if (exact < goal && cut_of_list<MASS>(c, row, exact, goal)) {
          *upto = end;
          if (!MASS) *above = 0, *upto = no_end();
          return kCut;
        }
      }
    }
  }
  cluster_barrier();  // the histograms and the list have been read
  clear_hist(c.hist);
  __syncthreads();
  return out;
}

// The cut of the shortest prefix whose value (its count: top-k; its mass: top-p)
// reaches a goal: k, or top_p of the mass inside the present cut. True when the row
// is finished. The histogram is clear on entry. All threads of the cluster call it,
// and every branch on the way to a barrier is the same for all of them.
template <bool MASS, typename P>
__device__ bool select(Cluster& c, const SampleParams& p, int row_b, Row& row, const P& part, uint32_t idx0, uint64_t k,
                       float top_p) {
  Shared& sh = c.sh;
  const int tid = threadIdx.x;
  uint64_t before = 0, goal = 0;              // the value of what lies above the range; the goal
  uint32_t lo = 0, hi = 0;                    // keys of the range, inclusive, after the first histogram
  int shift = 0;
  bool first = true;  // the first histogram is over Row::place, the others over the bits of the keys
  for (int pass = 0; pass < 6; ++pass) {  // at most 4 are needed: 2048 bins, then 11 bits of the key each
    part.each(row.alive, [&](float v, int i) {
      const uint32_t key = key_of(v);
      if (!(v >= row.alive) || (!first && (key < lo || key > hi)) || !row.inside(v, idx0 + i)) return;
      const int b = first ? (int)row.place(v) : (int)((hi - key) >> shift);
      const uint64_t mass = MASS ? row.weight_of(row.exponent(v)) : 1ull;
      if (mass) atomicAdd(&c.hist.bin[b], (unsigned long long)mass);
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
      klo = key_of(row.least((float)(f.bin + 1)));
      khi = f.bin ? key_of(row.least((float)f.bin)) - 1 : key_of(row.top);
    } else {
      khi = hi - ((uint32_t)f.bin << shift);
      klo = khi - lo > (1u << shift) - 1 ? khi - ((1u << shift) - 1) : lo;
    }
    const float least = key_value(klo), end = khi < key_of(row.top) ? key_value(khi + 1) : no_end();
    // how many elements there are: counted, or bounded by the least and the greatest mass that they may have
    const uint64_t w_lo = MASS ? row.weight(least) : 1, w_hi = MASS ? row.weight(key_value(khi)) : 1;
    const bool down = first && before + f.value <= kCand * w_lo;
    if (down || f.value <= kCand * w_hi) {
      collect(c, row, part, idx0, least, down ? no_end() : end, [](float, int) {});
      if (collected(c) <= (uint32_t)kCand) {
        if (down) {
          last_read(c, [&] { finish<!MASS>(sh, p, row_b, row, k, goal, top_p); });
          return true;
        }
        cut_of_list<MASS>(c, row, before, goal);
        return false;
      }
    }
    if (klo == khi) {
      // many equal keys: the goal's place among them, in index order
      const uint64_t g = w_lo, need = (goal - before + g - 1) / g;  // ties to keep, >= 1
      uint64_t ties = 0;
      part.each(least, [&](float v, int i) { ties += v == least && row.inside(v, idx0 + i); });
#pragma unroll
      for (int o = 16; o; o >>= 1) ties += __shfl_xor_sync(0xffffffffu, ties, o);
      // (a warp's block is contiguous: warps are in index order)
      uint64_t all;
      uint64_t tb = block_scan(sh, (tid & 31) == 0 ? ties : 0, &all);
      tb = __shfl_sync(0xffffffffu, tb, 0);
      const auto tslots = c.exchange(all, 0);
      for (int r = 0; r < c.rank; ++r) tb += tslots[r][0];
      if (tid == 0) sh.found[0] = ~0ull;
      __syncthreads();
      if (tb < need && need <= tb + ties) {
        const int i0 = (tid >> 5) * part.blk, lane = tid & 31;
        for (int i = i0; i < i0 + part.blk; i += 32) {
          const float4 q = part.four(i + lane);
          const int at = 4 * (i + lane);
          const bool is[4] = {q.x == least && row.inside(least, idx0 + at), q.y == least && row.inside(least, idx0 + at + 1),
                              q.z == least && row.inside(least, idx0 + at + 2),
                              q.w == least && row.inside(least, idx0 + at + 3)};
          int inc = is[0] + is[1] + is[2] + is[3];
          const int four = inc;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += up;
          }
          uint64_t at_tie = tb + inc - four;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (is[e] && ++at_tie == need) sh.found[0] = idx0 + at + e;
          tb += __shfl_sync(0xffffffffu, inc, 31);
        }
      }
      __syncthreads();
      const auto cut = c.exchange(sh.found[0], 0);
      for (int r = 0; r < c.size; ++r)
        if (cut[r][0] != ~0ull) {
          row.cut = least;
          row.cut_idx = (uint32_t)cut[r][0];
        }
      return false;
    }
    // many elements of unlike keys: another histogram over the bin's keys
    cluster_barrier();  // every CTA has read the histograms
    lo = klo;
    hi = khi;
    first = false;
    shift = max(0, 32 - __clz(hi - lo) - 11);  // hi - lo < 2^(32 - clz)
    clear_hist(c.hist);
    __syncthreads();
  }
  return false;
}

template <typename T, bool HELD>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const __grid_constant__ SampleParams p) {
  // the histogram when there are top_k or top_p, then the logits [chunk] when they are held
  extern __shared__ __align__(16) uint8_t dynamic[];
  __shared__ Shared sh;
  cluster_arrive_relaxed();  // matched by the wait before the first remote store
  uint32_t size;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(size));
  const bool hist = p.top_k || p.top_p;
  Cluster c{sh, *reinterpret_cast<Hist*>(dynamic), (int)cluster_ctarank(), (int)size, 0};
  const int b = blockIdx.x / size, tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const uint32_t idx0 = c.rank * p.chunk;
  Part<T, HELD> part;
  {
    const T* x = static_cast<const T*>(p.x) + (int64_t)b * p.ld;
    part.held = reinterpret_cast<float4*>(dynamic + (hist ? sizeof(Hist) : sizeof(Queue)));
    part.x = x + idx0;
    part.n = (int)min((int64_t)p.chunk, max((int64_t)0, (int64_t)p.V - idx0));
    part.blk = p.chunk / 4 / kWarps;
    const int groups = (part.blk + 32 * kGroup - 1) / (32 * kGroup);
    part.peak = reinterpret_cast<__nv_bfloat16*>(part.held) + w * groups * 32;
    part.hits = reinterpret_cast<uint16_t*>(part.held) + kThreads * groups + w * kHits;
    part.whole = reinterpret_cast<uintptr_t>(x) % (4 * sizeof(T)) == 0;  // (idx0 is a multiple of 4)
  }
  if (tid < 64) sh.exp2_64[tid] = exp2(tid / 64.0);
  if (hist) clear_hist(c.hist);
  pdl_launch_dependents();
  pdl_wait();
  const float temp = p.temp ? p.temp[b] : 1.0f;
  const int k = p.top_k ? p.top_k[b] : 0;
  const float tp = p.top_p ? p.top_p[b] : 1.0f;
  // the part's largest with the lowest index (NaN never wins)
  uint64_t best;
  {
    const int end = (w + 1) * part.blk;
    float top = -INFINITY;
    uint32_t at = idx0 + 4 * (w * part.blk + lane);
    constexpr int kAtOnce = kGroup;
    const float4 nothing = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    float4 q[kAtOnce], next[kAtOnce];
    auto load = [&](float4(&to)[kAtOnce], int i0) {
#pragma unroll
      for (int a = 0; a < kAtOnce; ++a) to[a] = i0 + 32 * a < end ? part.raw(i0 + 32 * a) : nothing;
    };
    load(next, w * part.blk + lane);
    for (int i0 = w * part.blk + lane; i0 < end; i0 += 32 * kAtOnce) {  // the next fours are on their way meanwhile
#pragma unroll
      for (int a = 0; a < kAtOnce; ++a) q[a] = next[a];
      load(next, i0 + 32 * kAtOnce);
      float peak = -INFINITY;
#pragma unroll
      for (int a = 0; a < kAtOnce; ++a) {
        const int i = i0 + 32 * a;
        if (HELD && i < end) part.held[i] = q[a];
        const float m = fmaxf(fmaxf(q[a].x, q[a].y), fmaxf(q[a].z, q[a].w));
        peak = fmaxf(peak, m);
        if (m > top) {  // (equal ones come later in the row)
          top = m;
          at = idx0 + 4 * i + (q[a].x == m ? 0 : q[a].y == m ? 1 : q[a].z == m ? 2 : 3);
        }
      }
      if (!HELD) part.peak[(i0 - w * part.blk - lane) / kGroup + lane] = __float2bfloat16_ru(peak);
    }
    part.largest = top;
    best = ((uint64_t)key_of(top) << 32) | (uint32_t)~at;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const uint64_t q = __shfl_xor_sync(0xffffffffu, best, o);
    best = q > best ? q : best;
  }
  if ((tid & 31) == 0) sh.warp[tid >> 5][0] = best;
  __syncthreads();
  for (int i = 0; i < kWarps; ++i) best = sh.warp[i][0] > best ? sh.warp[i][0] : best;
  // every CTA of the cluster is running: its shared memory may be written (one that has no logits comes here at once)
  __syncwarp();
  cluster_wait_acquire();
  {
    const auto s = c.exchange(best, 0);
    for (int r = 0; r < c.size; ++r) best = s[r][0] > best ? s[r][0] : best;
  }
  Row row;
  const uint32_t top_key = (uint32_t)(best >> 32), top_idx = ~(uint32_t)best;
  const bool none = top_key <= kNegInf;
  if (none || !(temp > 0.0f)) {  // nothing to draw from, or greedy
    if (c.rank == 0 && tid == 0) {
      const int32_t t = none ? 0 : (int32_t)top_idx;
      p.tok[b] = t;
      if (p.tok2) p.tok2[b] = t;
      if (p.logprob) p.logprob[b] = none ? __uint_as_float(0x7fc00000u) : 0.0f;
    }
    return;
  }
  row.top = key_value(top_key);
  row.m = (double)row.top;
  row.inv_t = 1.0 / (double)temp;
  row.bin_scale = (float)kBins / kSpan / temp;
  row.S = p.S;
  row.cut = -INFINITY;
  row.cut_idx = 0xffffffffu;
  row.table = sh.exp2_64;
  row.alive = row.least((float)kBins);
  row.min_e = -INFINITY;
  float least = row.alive;  // logits below are not kept
  {
    const float mp = p.min_p ? p.min_p[b] : 0.0f;
    if (mp > 0.0f) {
      row.min_e = fmin(log((double)mp), 0.0);
      // place() is within 2^-22 of the exact one, relative
      const float bound = (float)(-row.min_e * (kBins / kSpan)) * (1.0f + 0x1p-20f) + 0x1p-20f;
      if (bound < (float)kBins) least = row.least(bound);
    }
  }
  const bool ks = k > 0 && k < p.V;
  uint64_t above = 0;       // this warp's mass of the kept logits from `upto` on, once known
  float upto = no_end();
  if (ks) {
    // (more than the ranking can hold needs no try)
    if (k <= kCand && top_of_threads(c, p, b, row, part, idx0, (uint64_t)k, tp)) return;
    const Outcome o = cut_by_counts<false>(c, p, b, row, part, idx0, (uint64_t)k, tp, &above, &upto);
    if (o == kFinished || (o == kFailed && select<false>(c, p, b, row, part, idx0, (uint64_t)k, tp))) return;
  }
  if (tp < 1.0f) {
    if (ks) {
      __syncthreads();
      clear_hist(c.hist);
      __syncthreads();
    }
    const Outcome o = cut_by_counts<true>(c, p, b, row, part, idx0, 0, tp, &above, &upto);
    if (o == kFinished || (o == kFailed && select<true>(c, p, b, row, part, idx0, 0, tp))) return;
    if (o == kFailed || row.min_e > -INFINITY) above = 0, upto = no_end();
  }
  least = fmaxf(least, row.cut);
  // running masses in index order
  auto kept = [&](float v, int i) -> uint64_t {
    if (!(v >= least) || !row.inside(v, idx0 + i)) return 0ull;
    const double e = row.exponent(v);
    return e >= row.min_e ? row.weight_of(e) : 0ull;
  };
  uint64_t mine = lane == 0 ? above : 0;
  if (least == row.alive && row.cut == -INFINITY) {  // no filter: nearly all of them
    part.each(least, [&](float v, int) { mine += row.weight(v); });
  } else {  // few of them, in few lanes at a time: the others' lanes help
    float* queue = reinterpret_cast<Queue*>(dynamic)->of[w];
    int n = 0;  // in the queue, the same in every lane
    auto take = [&] {
      __syncwarp();
      n -= 32;
      if (n + lane >= 0) {
        const double e = row.exponent(queue[n + lane]);
        if (e >= row.min_e) mine += row.weight_of(e);
      }
      __syncwarp();
    };
    part.fours(least, [&](const float4& f, int at) {
      const float v[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool is = v[e] >= least && !(v[e] >= upto) && row.inside(v[e], idx0 + at + e);
        const unsigned are = __ballot_sync(0xffffffffu, is);
        if (is) queue[n + __popc(are & ((1u << lane) - 1))] = v[e];
        n += __popc(are);
      }
#pragma unroll 1
      while (n >= 32) take();
    });
    if (n > 0) take();
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  __syncthreads();
  if (lane == 0) sh.warp[w][0] = mine;
  __syncthreads();
  uint64_t cta = 0;
  for (int i = 0; i < kWarps; ++i) cta += sh.warp[i][0];
  const auto s = c.exchange(cta, 0);
  uint64_t z = 0, run = 0;
  for (int r = 0; r < c.size; ++r) {
    if (r < c.rank) run += s[r][0];
    z += s[r][0];
  }
  const uint64_t goal = goal_of_u(p.u[b], z);
  // the warp whose block holds the token; its rounds of 32 fours are shared out among all warps, and the one that has
  // the token in its rounds walks them
  if (!(run <= goal && goal < run + cta)) return;
  int of = 0;
  while (of + 1 < kWarps && goal >= run + sh.warp[of][0]) run += sh.warp[of++][0];
  const int rounds = part.blk / 32, each = (rounds + kWarps - 1) / kWarps;
  const int r0 = min(w * each, rounds), r1 = min(r0 + each, rounds);
  auto masses = [&](int r, float4& q, uint64_t(&v)[4]) {
    const int i = of * part.blk + 32 * r + lane;
    q = part.four(i);
    v[0] = kept(q.x, 4 * i);
    v[1] = kept(q.y, 4 * i + 1);
    v[2] = kept(q.z, 4 * i + 2);
    v[3] = kept(q.w, 4 * i + 3);
  };
  float4 q;
  uint64_t v[4], sum = 0;
#pragma unroll 1
  for (int r = r0; r < r1; ++r) {
    masses(r, q, v);
    sum += v[0] + v[1] + v[2] + v[3];
  }
  uint64_t inc = sum;
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) sh.warp[w][1] = sum;
  __syncthreads();
  for (int i = 0; i < w; ++i) run += sh.warp[i][1];
  if (!(run <= goal && goal < run + sum)) return;
#pragma unroll 1
  for (int r = r0; r < r1; ++r) {
    if (each > 1) {  // (else they are at hand)
      masses(r, q, v);
      inc = v[0] + v[1] + v[2] + v[3];
    }
    const uint64_t four = inc;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t up = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += up;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, run + inc > goal);
    if (hit) {
      if (lane == __ffs(hit) - 1) {
        const float logit[4] = {q.x, q.y, q.z, q.w};
        run += inc - four;
        bool done = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          run += v[e];
          if (!done && run > goal) {
            put_token(p, b, row, logit[e], idx0 + 4 * (of * part.blk + 32 * r + lane) + e, z);
            done = true;
          }
        }
      }
      return;
    }
    run += __shfl_sync(0xffffffffu, inc, 31);
  }
}

// dynamic shared memory with which a CTA has an SM to itself
constexpr int kAlone = 114 * 1024 - (int)sizeof(Shared);
}  // namespace

int sample_setup(DeviceInfo& d) {
  // a held part or the summary of the longest row, and the histogram
  constexpr int kMost = kHeld * 4 + kWarps * kHits * 2 + (int)sizeof(Hist);
  static_assert(BTF_SAMPLE_MAX_V / (4 * kGroup) * 2 <= kHeld * 4);
  if (kMost + (int)sizeof(Shared) + 1024 > d.optin_smem)
    return fail(BTF_ERR_UNSUPPORTED, "sample_kernel needs %d bytes of shared memory", kMost + (int)sizeof(Shared));
  for (const auto f : {sample_kernel<float, true>, sample_kernel<__half, true>, sample_kernel<__nv_bfloat16, true>,
                       sample_kernel<float, false>, sample_kernel<__half, false>, sample_kernel<__nv_bfloat16, false>}) {
    cudaError_t e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(f, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return cuda_fail(e, "sample_kernel attributes");
  }
  for (int i = 0; i < 5; ++i) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(1u << i);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kAlone;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = 1u << i;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&d.sample_clusters[i], sample_kernel<float, true>, &cfg) != cudaSuccess) {
      d.sample_clusters[i] = 0;
      cudaGetLastError();
    }
  }
  return BTF_OK;
}

cudaError_t launch_sample(const SampleArgs& a, cudaStream_t st) {
  SampleParams p{a.logits, a.ld, a.V, 0, 62, a.u, a.temperature, a.top_p, a.min_p, a.top_k, a.tokens, a.tokens2,
                 a.logprobs};
  int lg = 0;
  while ((1ll << lg) < a.V) ++lg;
  p.S = std::min(44, 62 - lg);
  // few rows: a CTA per kHeld logits or less, which stay in shared memory, and further
  // ones down to kLeast as long as every CTA has an SM of its own (one row of 128003:
  // top-p 27.1 -> 23.0 us with 16 CTAs for 8, no filter 15.1 -> 10.7; below 4096 the
  // barriers cost what is saved), which they then ask for (33 rows of 50257 with every
  // filter: 18.6 us, 23.3 two to an SM with others idle); more CTAs than are resident at
  // once (2 per SM): fewer and larger parts, read again
  const DeviceInfo* dev = current_device();
  if (!dev) return cudaErrorInitializationError;
  const int slots = 2 * dev->sm_count;
  auto alone = [&](int i) { return i < 5 && a.B <= dev->sample_clusters[i]; };  // 2^i CTAs a row, an SM each
  int size = 1, lg_size = 0;
  while (size < kMaxCluster && ((a.V + size - 1) / size > kHeld ||
                                ((a.V + size - 1) / size > kLeast && alone(lg_size + 1))))
    size *= 2, ++lg_size;
  bool held = (a.V + size - 1) / size <= kHeld;
  if ((int64_t)a.B * size > slots && size > 1) {
    held = false;
    while (size > 1 && (int64_t)a.B * size > slots) size /= 2, --lg_size;
  }
  constexpr int kStep = 4 * kThreads;
  p.chunk = ((a.V + size - 1) / size + kStep - 1) / kStep * kStep;
  const int groups = (p.chunk / 4 / kWarps + 32 * kGroup - 1) / (32 * kGroup);
  size_t smem = (held ? (size_t)p.chunk * 4 : ((size_t)groups * kThreads + kWarps * kHits) * 2) +
                      (a.top_k || a.top_p ? sizeof(Hist) : sizeof(Queue));
  if (alone(lg_size)) smem = std::max(smem, (size_t)kAlone);
  const auto kernel =
      a.type == BTF_F32   ? (held ? sample_kernel<float, true> : sample_kernel<float, false>)
      : a.type == BTF_F16 ? (held ? sample_kernel<__half, true> : sample_kernel<__half, false>)
                          : (held ? sample_kernel<__nv_bfloat16, true> : sample_kernel<__nv_bfloat16, false>);
  return launch_pdl_cluster(kernel, dim3((unsigned)(a.B * size)), dim3(kThreads), smem, st, size, p);
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
