// Attention of a few new tokens over rows of K and V, on the tcgen05 tensor cores:
// the kernel that btf_tree_attention and btf_prefix_attention share.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale q_i . k_j - m_i)
//
// over the cached rows and, among the tree's own rows, node i and its ancestors.
// The q-heads of a kv-head read the same K and V, so the n nodes x G heads of a
// kv-head are the rows of one matrix: 128 of them make the M side of the MMAs and
// every K and V row is read once for all of them.
//
// What bounds it: a tile of 64 rows of K and V is 256 D bytes and, whatever the
// number of q rows, 2 x 128 x 64 x D multiply-adds on the tensor core: at 6.5
// TB/s and 1.68 PFLOP/s over 148 SMs the bytes take 2.5 times as long as the MMAs.
// So up to 128 rows a kv-head the kernel is bound by the cache's bytes, and beyond
// that (more M tiles over the same cache, which then comes from L2) by the MMAs.
//
// Work: the 64-row tiles of all (sequence, kv-head) pairs, by their present
// lengths, in as many equal ranges as there are resident CTAs (per M tile: the
// CTAs of one range's M tiles read the same rows at the same time). A pair of
// several ranges is finished by a second kernel from its parts; a short cache, a
// long one and a ragged batch all fill the card. Warp 4 loads K and V tiles by TMA
// into a ring, warp 5 issues the MMAs, warps 0..3 hold one q row per thread:
//   S = Q K^T (64 columns of tensor memory, two of them in turn) -> registers,
//   mask, running maximum, p = 2^(s - m) -> 16 bits, the A operand of O += P V (from
//   the tensor memory of S, or shared memory; V as it lies: MN-major B).
// S of the next tile (the next two at D > 128) is computed during the softmax of this one. The maximum that p
// is taken against only moves when a row's grows by more than 2^8 (m then jumps and
// O is rescaled in tensor memory); p stays below 2^8, which the type holds, and
// the sum below it is exact in fp32 all the same.
// At D > 128 Q sits in tensor memory and P in shared memory: from shared memory a
// 128 x 64 x 16 MMA of Q K^T reads 6 KB in the 32 cycles that it takes, more than the
// 4 KB that shared memory gives, and S of tile j + 2 need not wait for P V of tile j.
//
// Measured (device time): 16 nodes x 24 heads of 256 over 4096 fp16 rows of 4
// kv-heads: 16.4 us (17 MB; the floor of a call, 1 node over 513 rows, is 10.1: two
// launches, lengths, q, K, V and the parts' way through memory one after another);
// 16 sequences of up to 8203 rows, 24 nodes, 32 and 8 heads of 128: 29.2 us, 3.3 TB/s;
// 1 node over 131072 rows 5.9 TB/s of K and V, 16 nodes 5.4; 64 nodes (three M tiles):
// 195 us, 1055 TFLOP/s (233 us, 883 TFLOP/s, call after call under the power cap). There a 64-row tile takes 1560 cycles, in which each SM gets its
// 64 KB of K and V (8.3 TB/s out of L2 for all) and moves 160 KB in shared memory; the
// MMAs alone take 1024. Two softmax threads per row gained nothing (202 us).
//
// p is rounded to the type of V (the MMA takes one type): eps / 2 per term, as much
// as the output's own rounding at most (the error against 64 bits of the cases above, of
// which the output's rounding is nearly all, grows by 1 to 10 %). fp16 p carry a factor 2^7, so that those
// down to 2^-32 of the largest still count. Scores, maxima, sums and O are fp32.
#pragma once
#include <algorithm>
#include <cmath>

#include "elem.cuh"
#include "tcgen05.cuh"

namespace btf {
namespace {

using namespace tc;

constexpr int kTile = 64;  // rows of K and V per tile
constexpr int kRowsM = 128;
constexpr int kThreads = 192;
constexpr uint64_t kWaitNs = 1000000000ull;
constexpr float kLag = 8.0f;  // log2 of how far a row's maximum may run ahead of m

template <int DP>  // D padded to whole 128-byte swizzle rows
struct Cfg {
  static constexpr int kBlocks = DP / 64;          // 64-column blocks
  // Q in tensor memory and P in shared memory [128 rows][128 B] x 2, or Q in shared
  // memory [block][128 rows][128 B] and P in S's tensor memory; SW128
  static constexpr bool kWide = DP > 128;
  static constexpr int kStage = kTile * DP * 2;    // [block][64 rows][128 B], SW128
  // one CTA per SM above 128 (its O takes half of tensor memory), two below: each
  // SM has 128 KB of copies in flight or more
  static constexpr int kStages = DP == 256 ? 5 : DP == 192 ? 7 : DP == 128 ? 4 : 9;
  static constexpr int kTmem = DP <= 128 ? 256 : 512;  // O: DP columns; S (P): 2 x 64; Q: DP / 2
  static constexpr int kPerSm = DP <= 128 ? 2 : 1;
  // a warp's 32 rows on their way between memory and tensor memory, 128 bytes of each, padded by 16
  static constexpr int kStageRow = 32 * 4 + 16, kOutWarp = 32 * kStageRow;
  static constexpr int kQBytes = kWide ? 0 : kRowsM * DP * 2;  // shares its place with the rows' way out
  static constexpr int kOffP = ((4 * kOutWarp > kQBytes ? 4 * kOutWarp : kQBytes) + 1023) / 1024 * 1024;
  static constexpr int kPBytes = kRowsM * kTile * 2;
  static constexpr int kOffRing = kOffP + (kWide ? 2 * kPBytes : 0);
  static constexpr int kOffMisc = kOffRing + kStages * kStage;
  static constexpr int kSmem = 1024 + kOffMisc + 512;
};

struct AttnParams {
  const void *q, *v;
  void* o;
  int64_t q_batch, q_node, q_head, kv_batch, kv_row, kv_head, o_batch, o_node, o_head;
  int B, n, H, HK, D, n_ctx, mtiles, ranges;
  int b_mul, h_mul;  // 0: every sequence / kv-head has the same K and V
  const int32_t *lens, *parents, *counts;
  float scale2;     // |scale| log2(e), at least 2^-100 (0 times the -inf of a masked score would be NaN)
  uint32_t q_flip;  // sign bits of two q when scale < 0
  int32_t* first;   // workspace: the table that the segments leave for the join
  float* part;      // rows of parts: [..][D]
  float* ml;        // their (m, l): [..][2]
  int* err;
};

// A sequence's nodes, cached rows and tiles.
struct Seq {
  int count, len, tiles;
  Seq() = default;
  __device__ __forceinline__ Seq(const AttnParams& p, int b) {
    count = p.counts ? min(max(p.counts[b], 0), p.n) : p.n;
    len = max(0, min(p.lens[b], p.n_ctx - count));
    tiles = count ? (len + count + kTile - 1) / kTile : 0;
  }
};

template <int N>
struct AttnMaps {
  CUtensorMap m[N];  // K and V, in pairs
};
// A row of a segment: whose it is. live: not padding.
struct RowPlace {
  int b, node, head;
  bool live;
};

// The segments of a CTA's range: runs of tiles of one (sequence, kv-head).
//
// Up to 32 sequences with fewer pairs than ranges: every pair is cut into its own
// number of equal ranges, n_b = ceil(tiles / per) with the least `per` that fits, and a
// CTA has one segment (a second one costs its q and its way out again, about 5 tiles
// of time: 1 x 1 node over 513 rows took 15.5 us with ranges across pairs, 12.0
// without; the search for `per` is 0.4 us of it, and left out for equal lengths). Otherwise the line of all tiles is cut into equal ranges.
// Both sides, own ranges and the line, in us for 8 nodes of 32 q-heads over 8 kv-heads: D = 128, 512 rows 11.8 and 11.8
// (40 pairs), 12.6 and 15.7 (80), 15.9 and 19.8 (240); 8192 rows 59 and 63 (80), 127 and 112 (160), 156 and 167 (240).
// D = 256, 512 rows 21.9 and 24.2 (80), 22.5 and 26.4 (128); 8192 rows 60 and 66 (40), 133 and 116 (80), 164 and 175 (128).
// So the line is up to 13 % ahead just above half as many pairs as ranges over long caches, where each pair has one
// range and nearly half of the CTAs none, and behind elsewhere. 32 sequences are what a warp works out at once, a lane
// each; what the 33rd of one kv-head costs: D = 128, 4096 rows 19.9 -> 20.6, D = 256 33.5 -> 39.1, 600 rows 15.2 -> 20.2.
//
// A pair on the line has `over` units in front of its tiles, the time of its q and its way out in tiles (0 where pairs
// are few and long): with short pairs, equal numbers of tiles alone give one range many pairs and many times the work.
//
// The table for the join: each sequence's first range, or first unit on the line; then units per range, and which of the
// two it is. The parts of a cut pair: two to a range, 1 for the pair whose first tile is in it.
struct Segments {
  const AttnParams& p;
  const int ranges, over, mt, range;
  int b, kvh, tile, nt;         // the present one
  int left;                     // units behind it
  Seq seq;
  // M tile block % mtiles of range block / mtiles (block < 0: no segment). Warp-uniform; every warp works it out for
  // itself. Writes the workspace's table when `table`.
  __device__ __forceinline__ Segments(const AttnParams& p_, int block, int ranges_, int over_, bool table)
      : p(p_), ranges(ranges_), over(over_), mt(block % p_.mtiles), range(block / p_.mtiles), b(0), kvh(0), tile(0), nt(0), left(0) {
    if (block < 0) return;
    const int lane = threadIdx.x & 31;
    Seq mine;  // the lane's sequence of the 32 from b0
    auto load = [&](int b0) {
      mine.count = mine.len = mine.tiles = 0;
      if (b0 + lane < p.B) mine = Seq(p, b0 + lane);
    };
    auto up_to = [&](int t) {  // the sum of the lanes up to this one
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int q = __shfl_up_sync(0xffffffffu, t, o);
        if (lane >= o) t += q;
      }
      return t;
    };
    // the sequence of the 32 from b0 in whose share of a line (up to `t` for each lane) `at` lies
    auto pick = [&](int b0, int t, int* at) -> bool {
      const unsigned in = __ballot_sync(0xffffffffu, t > *at);
      if (!in) return false;
      const int l = __ffs(in) - 1, before = __shfl_sync(0xffffffffu, t, max(l - 1, 0));
      b = b0 + l;
      *at -= l ? before : 0;
      seq.count = __shfl_sync(0xffffffffu, mine.count, l);
      seq.len = __shfl_sync(0xffffffffu, mine.len, l);
      seq.tiles = __shfl_sync(0xffffffffu, mine.tiles, l);
      return true;
    };
    load(0);
    const int pairs = p.HK * __popc(__ballot_sync(0xffffffffu, mine.tiles > 0));
    if (p.B <= 32 && pairs <= ranges) {
      const int longest = __reduce_max_sync(0xffffffffu, mine.tiles);
      int per = 1;
      if (__all_sync(0xffffffffu, mine.tiles == 0 || mine.tiles == longest)) {  // (all of one length: no search)
        const int each = ranges / max(pairs, 1);
        per = max(1, (longest + each - 1) / each);
      } else {
        const int total = p.HK * __reduce_add_sync(0xffffffffu, mine.tiles);
        per = max(1, (total + ranges - 1) / ranges);
        // sum ceil(tiles / per) <= total / per + pairs
        int most = pairs < ranges ? max(per, (total + ranges - pairs - 1) / (ranges - pairs)) : max(1, total);
        while (per < most) {
          const int mid = (per + most) / 2;
          if (p.HK * __reduce_add_sync(0xffffffffu, (mine.tiles + mid - 1) / mid) <= ranges) most = mid;
          else per = mid + 1;
        }
      }
      const int n = (mine.tiles + per - 1) / per, t = up_to(n * p.HK);
      if (table && lane < p.B) p.first[lane] = t - n * p.HK;
      if (table && lane == 0) p.first[p.B] = per, p.first[p.B + 1] = 1;
      int at = range;
      if (!pick(0, t, &at)) return;
      const int ns = (seq.tiles + per - 1) / per, part = at % ns;
      kvh = at / ns;
      tile = (int)((int64_t)part * seq.tiles / ns);
      nt = (int)((int64_t)(part + 1) * seq.tiles / ns) - tile;
      return;
    }
    auto units = [&]() { return mine.tiles ? (mine.tiles + over) * p.HK : 0; };
    int total = 0, t = 0;
    for (int b0 = 0; b0 < p.B; b0 += 32) {
      load(b0);
      t = up_to(units());
      if (table && b0 + lane < p.B) p.first[b0 + lane] = total + t - units();
      total += __shfl_sync(0xffffffffu, t, 31);
    }
    const int per = max(1, (total + ranges - 1) / ranges);
    if (table && lane == 0) p.first[p.B] = per, p.first[p.B + 1] = 0;
    if ((int64_t)range * per >= total) return;
    int start = range * per;
    left = min(per, total - start);
    for (int b0 = 0;; b0 += 32) {  // the sequence that the range starts in
      load(b0);
      t = up_to(units());
      if (pick(b0, t, &start)) break;
      start -= __shfl_sync(0xffffffffu, t, 31);
    }
    kvh = start / (seq.tiles + over);
    take(start % (seq.tiles + over));
    if (nt == 0) next();  // (the range begins with the end of a pair's units in front)
  }
  // The present pair from its unit `at`.
  __device__ __forceinline__ void take(int at) {
    const int to = min(at + left, seq.tiles + over);
    left -= to - at;
    tile = max(0, at - over);
    nt = max(0, to - over) - tile;
  }
  __device__ __forceinline__ bool any() const { return nt > 0; }
  __device__ __forceinline__ void next() {
    nt = 0;
    while (nt == 0 && left > 0) {
      if (++kvh == p.HK) {
        kvh = 0;
        do seq = Seq(p, ++b);
        while (seq.tiles == 0);
      }
      take(0);
    }
  }
  __device__ __forceinline__ int rows() const { return min(kRowsM, seq.count * (p.H / p.HK) - mt * kRowsM); }
  __device__ __forceinline__ int plane_b() const { return b * p.b_mul; }
  __device__ __forceinline__ int plane_h() const { return kvh * p.h_mul; }
  __device__ __forceinline__ RowPlace place_of(int r) const {
    const int G = p.H / p.HK, rr = mt * kRowsM + r;
    const bool live = r < rows();
    return {b, live ? rr / G : 0, kvh * G + (live ? rr % G : 0), live};
  }
  // By the table: the first range of a (sequence, kv-head), and their number.
  static __device__ __forceinline__ int ranges_of(const AttnParams& p, int over, const Seq& seq, int b, int kvh, int* n) {
    const int per = p.first[p.B], first = p.first[b];
    if (p.first[p.B + 1]) {
      *n = (seq.tiles + per - 1) / per;
      return first + kvh * *n;
    }
    const int t0 = first + kvh * (seq.tiles + over) + over, t1 = t0 + seq.tiles - 1, r0 = t0 / per;
    *n = t1 / per - r0 + 1;
    return r0;
  }
};

// Itself and its ancestors, as bits, for this lane's nodes `lane` and `lane + 32`: pointer doubling over the
// parents (a parent that is not an earlier node hangs on the cache).
__device__ __forceinline__ void tree_masks(const int32_t* parents, int n, uint64_t (&m)[2]) {
  const int lane = threadIdx.x & 31;
  int jump[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int j = lane + 32 * r, pj = j < n ? parents[j] : -1;
    jump[r] = pj >= 0 && pj < j ? pj : -1;
    m[r] = 1ull << j;
  }
  for (int reach = 1; reach < n; reach *= 2) {
    uint64_t nm[2];
    int nj[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int a = jump[r], src = a & 31;
      const uint64_t m0 = __shfl_sync(0xffffffffu, m[0], src), m1 = __shfl_sync(0xffffffffu, m[1], src);
      const int j0 = __shfl_sync(0xffffffffu, jump[0], src), j1 = __shfl_sync(0xffffffffu, jump[1], src);
      nm[r] = m[r] | (a < 0 ? 0ull : a < 32 ? m0 : m1);
      nj[r] = a < 0 ? -1 : a < 32 ? j0 : j1;
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) m[r] = nm[r], jump[r] = nj[r];
  }
}

__device__ __forceinline__ void st_if(void* to, uint4 v, bool on) {  // predicated: no branch per store
  asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %5, 0;\n @p st.global.v4.u32 [%0], {%1, %2, %3, %4};\n}\n" ::"l"(to),
               "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w), "r"((int)on)
               : "memory");
}
__device__ __forceinline__ float ex2(float x) {  // 2^x, 2 ulp; 0 below 2^-126
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {  // one conversion for both
  if constexpr (std::is_same_v<T, __half>) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
// Shared memory behind the ring. What is signalled once per tile has two barriers,
// used in turn: a wait for tile t may begin while t - 1 is under way (its parity
// on one barrier would read as t's done), and t - 2 is done by then.
struct Misc {
  uint64_t full[10], empty[10], s_full[2], s_free[2], p_ready[2], pv_done[2], q_ready, final;  // mbarriers
  unsigned long long bad;  // nodes with an infinity or NaN in V
  uint32_t tmem;
  int abort;
};
static_assert(sizeof(Misc) <= 512);

// The ring's order within a segment of nt tiles: K runs AHEAD tiles before V, as
// the MMAs take them: K_0 .. K_(AHEAD - 1), then K_(j + AHEAD), V_j for j = 0, 1, ...
template <int AHEAD>
__device__ __forceinline__ int item_of_k(int j) { return j < AHEAD ? j : 2 * j - AHEAD; }
template <int AHEAD>
__device__ __forceinline__ int item_of_v(int j, int nt) { return min(j + AHEAD + 1, nt) + j; }

// W: a CTA's segments, where their rows of q lie and where their parts go (TreeSegments of tree_attn.cu, PrefixSegments
// of prefix_attn.cu).
template <typename T, int DP, typename W>
__global__ void __launch_bounds__(kThreads, Cfg<DP>::kPerSm)
    attn_kernel(const __grid_constant__ AttnMaps<W::kMaps> maps, const __grid_constant__ typename W::Params p) {
  using C = Cfg<DP>;
  constexpr int kAhead = C::kWide ? 2 : 1;
  constexpr bool kBf16 = std::is_same_v<T, __nv_bfloat16>;
  constexpr float kBias = kBf16 ? 0.0f : 7.0f;  // fp16 p times 2^7 (below 2^8 * 2^7)
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw), sbase = (raw + 1023) & ~1023u;
  uint8_t* smem = smem_raw + (sbase - raw);
  Misc& ms = *reinterpret_cast<Misc*>(smem + C::kOffMisc);
  volatile int* abort_flag = &ms.abort;
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  if (warp == 5) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ms.tmem)),
                 "r"((uint32_t)C::kTmem)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (warp == 4 && lane == 0) {
#pragma unroll
    for (int i = 0; i < W::kMaps; ++i) prefetch_map(&maps.m[i]);
  }
  if (tid == 0) {
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(smem_u32(&ms.full[i]), 1);
      mbar_init(smem_u32(&ms.empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&ms.s_full[i]), 1);
      mbar_init(smem_u32(&ms.s_free[i]), 4);
      mbar_init(smem_u32(&ms.p_ready[i]), 4);
      mbar_init(smem_u32(&ms.pv_done[i]), 1);
    }
    mbar_init(smem_u32(&ms.q_ready), 4);
    mbar_init(smem_u32(&ms.final), 1);
    ms.bad = 0;
    ms.abort = 0;
    fence_mbar_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, ms.tmem, 0), tmem_s = tmem + DP, tmem_q = tmem + DP + 2 * kTile;
  pdl_launch_dependents();
  pdl_wait();

  // bounded wait; false (and the abort flag set) on a time-out or after another role's time-out
  auto wait = [&](const uint64_t& bar, uint32_t parity) -> bool {
    const uint32_t a = smem_u32(&bar);
    if (mbar_try_wait(a, parity)) return true;
    if (*abort_flag) return false;
    if (mbar_wait_bounded(a, parity, kWaitNs)) return true;
    atomicCAS(p.err, 0, kErrWaitTimeout);
    *abort_flag = 1;
    return false;
  };
  // the same for a whole warp: true in every lane, or in none
  auto warp_wait = [&](const uint64_t& bar, uint32_t parity) -> bool {
    return __all_sync(0xffffffffu, wait(bar, parity));
  };
  W sg(p, warp == 0);
  if (warp == 4) {
    // ---------------------------------------------------------- K and V tiles
    if (lane == 0) {
      int i = 0;
      bool ok = true;
      for (; ok && sg.any(); sg.next()) {
        if (sg.rows() <= 0) continue;
        const int zb = sg.plane_b(), zh = sg.plane_h(), map = sg.map();
        auto load = [&](const CUtensorMap* m, int j) -> bool {
          const int s = i % C::kStages;
          if (i >= C::kStages && !wait(ms.empty[s], (uint32_t)((i / C::kStages - 1) & 1))) return false;
          const uint32_t bar = smem_u32(&ms.full[s]), dst = sbase + C::kOffRing + s * C::kStage;
          mbar_expect_tx(bar, C::kStage);
#pragma unroll
          for (int c = 0; c < C::kBlocks; ++c)
            tma_load_4d(dst + c * kTile * 128, m, c * 64, (sg.tile + j) * kTile, zh, zb, bar);
          ++i;
          return true;
        };
        for (int j = -kAhead; ok && j < sg.nt; ++j) {
          if (j + kAhead < sg.nt) ok = load(&maps.m[map], j + kAhead);
          if (ok && j >= 0) ok = load(&maps.m[map + 1], j);
        }
      }
      // after a time-out, leave no copy in flight into this CTA's shared memory (bounded)
      if (!ok || *abort_flag)
        for (int k = max(0, i - C::kStages); k < i; ++k)
          mbar_wait_bounded(smem_u32(&ms.full[k % C::kStages]), (uint32_t)((k / C::kStages) & 1), kWaitNs / 10);
    }
  } else if (warp == 5) {
    // ---------------------------------------------------------- MMAs
    constexpr uint32_t kQk = idesc_f16(kBf16, false, kRowsM, kTile), kPv = idesc_f16(kBf16, true, kRowsM, DP);
    const uint64_t qd = smem_desc_sw128(sbase);
    int g = 0;  // tiles before the segment's
    // S of the segment's tile j
    auto qk = [&](int j) -> bool {
      const int i = 2 * g + item_of_k<kAhead>(j), s = i % C::kStages;
      if (!warp_wait(ms.full[s], (uint32_t)((i / C::kStages) & 1))) return false;
      // S of tile j - 2 is in registers; where P lies in it, P has been read (a segment's first two tiles come after
      // everything of the one before)
      if (j >= 2 && !warp_wait(C::kWide ? ms.s_free[(g + j) & 1] : ms.pv_done[(g + j) & 1],
                               (uint32_t)(((g + j - 2) >> 1) & 1)))
        return false;
      tc_fence_after();
      const uint64_t kd = smem_desc_sw128(sbase + C::kOffRing + s * C::kStage);
      const uint32_t d = tmem_s + ((g + j) & 1) * kTile;
      if (elect_one()) {
#pragma unroll 1
        for (int blk = 0; blk < C::kBlocks; ++blk) {  // (a short loop: cold code costs a small call its fetch)
          const uint64_t kb = kd + (blk * kTile * 128 >> 4);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            if constexpr (C::kWide) mma_f16_ts(d, tmem_q + blk * 32 + c * 8, kb + (c * 32 >> 4), kQk, blk > 0 || c > 0);
            else mma_f16_ss(d, qd + ((blk * kRowsM * 128 + c * 32) >> 4), kb + (c * 32 >> 4), kQk, blk > 0 || c > 0);
          }
        }
        mma_commit(smem_u32(&ms.s_full[(g + j) & 1]));
        mma_commit(smem_u32(&ms.empty[s]));
      }
      __syncwarp();
      return true;
    };
    bool ok = true;
    int n = 0;
    for (; ok && sg.any(); sg.next()) {
      if (sg.rows() <= 0) continue;
      ok = warp_wait(ms.q_ready, (uint32_t)(n++ & 1));
      for (int j = -kAhead; ok && j < sg.nt; ++j) {
        if (j + kAhead < sg.nt && !(ok = qk(j + kAhead))) break;
        if (j < 0) continue;
        const int t = g + j, i = 2 * g + item_of_v<kAhead>(j, sg.nt), s = i % C::kStages;
        ok = warp_wait(ms.full[s], (uint32_t)((i / C::kStages) & 1)) &&
             warp_wait(ms.p_ready[t & 1], (uint32_t)((t >> 1) & 1));
        if (!ok) break;
        tc_fence_after();
        const uint64_t vd = smem_desc_mn_sw128(sbase + C::kOffRing + s * C::kStage, kTile * 128);
        if (elect_one()) {
#pragma unroll
          for (int c = 0; c < kTile / 16; ++c) {
            const uint64_t vc = vd + (c * 2048 >> 4);
            if constexpr (C::kWide)
              mma_f16_ss(tmem, smem_desc_sw128(sbase + C::kOffP + (t & 1) * C::kPBytes + c * 32), vc, kPv, j > 0 || c > 0);
            else mma_f16_ts(tmem, tmem_s + (t & 1) * kTile + c * 8, vc, kPv, j > 0 || c > 0);
          }
          mma_commit(smem_u32(&ms.pv_done[t & 1]));
          mma_commit(smem_u32(&ms.empty[s]));
        }
        __syncwarp();
      }
      g += sg.nt;
    }
    if (elect_one()) mma_commit(smem_u32(&ms.final));  // completes when every MMA issued above has finished
    __syncwarp();
    mbar_wait_bounded(smem_u32(&ms.final), 0, kWaitNs);
    __syncwarp();
  } else {
    // ---------------------------------------------------------- softmax, one row per thread
    const uint32_t lanes = (uint32_t)(warp * 32) << 16;
    uint8_t* stage = smem + warp * C::kOutWarp;
    int g = 0;
    for (; sg.any(); sg.next()) {
      const int rows = sg.rows();
      if (rows <= 0) continue;
      const int active = (rows + 31) >> 5;  // warps with rows; the others only keep step
      const Seq& seq = sg.seq;
      const int r = tid;
      const typename W::Place at = sg.place(r, warp < active);  // (warp-uniform condition)
      const bool live = at.live;
      // the warp's q rows: 4 rows of 128 bytes at a time, 8 lanes each
      if (warp < active) {
        const T* q = static_cast<const T*>(p.q);
        const int64_t qo = live ? at.b * p.q_batch + at.node * p.q_node + at.head * p.q_head : -1;
        uint4 x[C::kBlocks][8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int64_t from = __shfl_sync(0xffffffffu, qo, k * 4 + (lane >> 3));
#pragma unroll
          for (int c = 0; c < C::kBlocks; ++c) {
            const int col = c * 64 + (lane & 7) * 8;
            x[c][k] = from >= 0 && col < p.D ? *reinterpret_cast<const uint4*>(q + from + col) : make_uint4(0, 0, 0, 0);
          }
        }
#pragma unroll
        for (int c = 0; c < C::kBlocks; ++c) {
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int row = k * 4 + (lane >> 3);
            uint4 v = x[c][k];
            v.x ^= p.q_flip, v.y ^= p.q_flip, v.z ^= p.q_flip, v.w ^= p.q_flip;
            uint8_t* to = C::kWide ? stage + row * C::kStageRow + (lane & 7) * 16
                                   : smem + c * (kRowsM * 128) + (warp * 32 + row) * 128 + (((lane & 7) ^ (row & 7)) << 4);
            *reinterpret_cast<uint4*>(to) = v;
          }
          if constexpr (C::kWide) {
            __syncwarp();
            uint32_t w[32];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const uint4 v = *reinterpret_cast<const uint4*>(stage + lane * C::kStageRow + i * 16);
              w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
            }
            __syncwarp();
            tmem_st32(tmem_q + c * 32 + lanes, w);
          }
        }
        if constexpr (C::kWide) tmem_wait_st();
        else fence_proxy_async_smem();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&ms.q_ready));
      uint64_t mask = 0;
      if (warp < active && sg.tree()) {
        uint64_t mm[2];
        tree_masks(p.parents + (int64_t)sg.b * p.n, seq.count, mm);
        const uint64_t m0 = __shfl_sync(0xffffffffu, mm[0], at.node & 31), m1 = __shfl_sync(0xffffffffu, mm[1], at.node & 31);
        if (live) mask = at.node < 32 ? m0 : m1;
      }
      float m = -INFINITY, l = 0.f;
      bool ok = true;
      for (int j = 0; j < sg.nt; ++j) {
        const int t0 = (sg.tile + j) * kTile, t = g + j;
        if (!(ok = warp_wait(ms.s_full[t & 1], (uint32_t)((t >> 1) & 1)))) break;
        if (warp < active) {
          tc_fence_after();
          const uint32_t ts = tmem_s + (t & 1) * kTile + lanes;
          uint32_t s0[32], s1[32];
          tmem_ld32(ts, s0);
          tmem_ld32(ts + 32, s1);
          tmem_wait_ld(s0);
          tmem_wait_ld(s1);
          if constexpr (C::kWide) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&ms.s_free[t & 1]));
          }
          if (t0 + kTile > seq.len) {
            // the tile reaches the tree's rows: what this row sees of it, as bits
            const int d = seq.len - t0;  // cached rows in the tile; below 0: it begins at node -d
            const uint64_t vis = d >= 0 ? ((1ull << d) - 1) | (mask << d) : mask >> -d;
            const uint32_t lo = (uint32_t)vis, hi = (uint32_t)(vis >> 32);
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              if (!((lo >> i) & 1)) s0[i] = 0xff800000u;
              if (!((hi >> i) & 1)) s1[i] = 0xff800000u;
            }
          }
          float mq[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int i = 0; i < 32; ++i)
            mq[i & 3] = fmaxf(mq[i & 3], fmaxf(__uint_as_float(s0[i]), __uint_as_float(s1[i])));
          const float mx = fmaxf(fmaxf(mq[0], mq[1]), fmaxf(mq[2], mq[3])) * p.scale2;
          if (__any_sync(0xffffffffu, mx > m + kLag)) {
            const float mn = fmaxf(m, mx), f = m == -INFINITY ? 0.f : ex2(m - mn);
            m = mn;
            l *= f;
            if (j > 0) {
              if (!(ok = warp_wait(ms.pv_done[(t - 1) & 1], (uint32_t)(((t - 1) >> 1) & 1)))) break;
              tc_fence_after();
#pragma unroll 1
              for (int c = 0; c < DP / 32; ++c) {
                uint32_t o[32];
                tmem_ld32(tmem + c * 32 + lanes, o);
                tmem_wait_ld(o);
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                tmem_st32(tmem + c * 32 + lanes, o);
              }
              tmem_wait_st();
            }
          }
          const float sub = kBias - (m == -INFINITY ? 0.f : m);
          const float2 sc2 = make_float2(p.scale2, p.scale2), sub2 = make_float2(sub, sub);
          float2 la = make_float2(0.f, 0.f), lb = la;
          // (word i of P over s0[i]: the elements that make it have been read)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float2 a = __ffma2_rn(make_float2(__uint_as_float(s0[2 * i]), __uint_as_float(s0[2 * i + 1])), sc2, sub2);
            a = make_float2(ex2(a.x), ex2(a.y));
            la = __fadd2_rn(la, a);
            s0[i] = pack2<T>(a.x, a.y);
          }
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float2 a = __ffma2_rn(make_float2(__uint_as_float(s1[2 * i]), __uint_as_float(s1[2 * i + 1])), sc2, sub2);
            a = make_float2(ex2(a.x), ex2(a.y));
            lb = __fadd2_rn(lb, a);
            s0[16 + i] = pack2<T>(a.x, a.y);
          }
          l += (la.x + la.y) + (lb.x + lb.y);
          if constexpr (C::kWide) {
            // the buffer's last reader is P V of tile t - 2
            if (j >= 2 && !(ok = warp_wait(ms.pv_done[t & 1], (uint32_t)(((t - 2) >> 1) & 1)))) break;
            uint8_t* ps = smem + C::kOffP + (t & 1) * C::kPBytes + r * 128;
#pragma unroll
            for (int i = 0; i < 8; ++i)
              *reinterpret_cast<uint4*>(ps + ((i ^ (r & 7)) << 4)) =
                  make_uint4(s0[4 * i], s0[4 * i + 1], s0[4 * i + 2], s0[4 * i + 3]);
            fence_proxy_async_smem();
          } else {
            tmem_st32(ts, s0);
            tmem_wait_st();
          }
        } else if (C::kWide) {
          if (lane == 0) mbar_arrive(smem_u32(&ms.s_free[t & 1]));
          // as the others: nobody is two tiles ahead on p_ready
          if (j >= 2 && !(ok = warp_wait(ms.pv_done[t & 1], (uint32_t)(((t - 2) >> 1) & 1)))) break;
        }
        if (t0 + kTile > seq.len) {
          // V rows behind the last node would meet p = 0, and so would a node's row for
          // those that do not see it: 0 x NaN. The former are zeroed; of the latter,
          // infinities and NaN are, and added at the end for those that see them.
          const int i = 2 * g + item_of_v<kAhead>(j, sg.nt), s = i % C::kStages;
          if (!(ok = warp_wait(ms.full[s], (uint32_t)((i / C::kStages) & 1)))) break;
          uint8_t* vs = smem + C::kOffRing + s * C::kStage;
          const int from = max(0, seq.len - t0), gone = max(0, min(kTile, seq.len + seq.count - t0));
          constexpr int kWords = DP / 8;  // 16-byte words of a row
          auto at = [&](int e) {
            const int row = e / kWords, c = e % kWords;
            return reinterpret_cast<uint4*>(vs + (c >> 3) * (kTile * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4));
          };
          for (int e = gone * kWords + tid; e < kTile * kWords; e += 128) *at(e) = make_uint4(0, 0, 0, 0);
#pragma unroll 2
          for (int e = from * kWords + tid; e < gone * kWords; e += 128) {
            const uint4 v = *at(e);
            constexpr uint32_t kExp = kBf16 ? 0x7f80u : 0x7c00u;
            uint32_t w[4] = {v.x, v.y, v.z, v.w};
            bool any = false;
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              if ((w[x] & kExp) == kExp) w[x] &= 0xffff0000u, any = true;
              if (((w[x] >> 16) & kExp) == kExp) w[x] &= 0xffffu, any = true;
            }
            if (any) {
              *at(e) = make_uint4(w[0], w[1], w[2], w[3]);
              atomicOr(&ms.bad, 1ull << (t0 + e / kWords - seq.len));
            }
          }
          fence_proxy_async_smem();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&ms.p_ready[t & 1]));
      }
      g += sg.nt;
      ok = ok && warp_wait(ms.pv_done[(g - 1) & 1], (uint32_t)(((g - 1) >> 1) & 1));
      // every warp's part of `bad` is in, and the warps agree on whether all went well
      int all_ok;
      asm volatile(
          "{\n .reg .pred p, q;\n setp.ne.b32 p, %1, 0;\n bar.red.and.pred q, 2, 128, p;\n selp.b32 %0, 1, 0, q;\n}\n"
          : "=r"(all_ok)
          : "r"((int)ok)
          : "memory");
      if (!all_ok) break;
      // ---------------------------------------------------------- the output rows, or this range's part of them
      if (warp < active) {
        tc_fence_after();
        const bool whole = sg.whole();
        const float inv = whole ? 1.0f / l : 1.0f;
        const int64_t slot = sg.slot();  // its first row among the parts'
        const uint64_t bad = ms.bad & mask;
        // where this lane's row goes (the lanes ask each other), or the first of its words of the parts
        const int64_t to = at.b * p.o_batch + at.node * p.o_node + at.head * p.o_head;
        float* part = p.part + (slot + warp * 32 + (lane >> 3)) * p.D + (lane & 7) * 4;
        const int left4 = rows - warp * 32 - (lane >> 3);
        uint8_t* mine = stage + lane * C::kStageRow;
        // 32 columns of the warp's rows, through shared memory: rows leave as whole 16-byte words of consecutive lanes
        auto emit = [&](int c, uint32_t (&o)[32]) {
          const int cols = p.D - c * 32;  // a multiple of 8
          if (cols <= 0) return;
#pragma unroll 1
          for (uint64_t left = bad; left; left &= left - 1) {
            const T* vr = static_cast<const T*>(p.v) + sg.b * p.kv_batch + sg.kvh * p.kv_head +
                          (int64_t)(seq.len + __ffsll((long long)left) - 1) * p.kv_row + c * 32;
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const float x = i < cols ? to_f32(vr[i]) : 0.f;
              if (!(fabsf(x) < INFINITY)) o[i] = __float_as_uint(__uint_as_float(o[i]) + x);
            }
          }
          __syncwarp();
          if (whole) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t w[4];
#pragma unroll
              for (int e = 0; e < 4; ++e)
                w[e] = pack2<T>(__uint_as_float(o[i * 8 + 2 * e]) * inv, __uint_as_float(o[i * 8 + 2 * e + 1]) * inv);
              reinterpret_cast<uint4*>(mine)[i] = make_uint4(w[0], w[1], w[2], w[3]);
            }
            __syncwarp();
#pragma unroll
            for (int k = 0; k < 4; ++k) {  // 8 rows of 64 bytes at a time
              const int row = k * 8 + (lane >> 2), x = lane & 3;
              const int64_t at = __shfl_sync(0xffffffffu, to, row);
              st_if(static_cast<T*>(p.o) + at + c * 32 + x * 8,
                    *reinterpret_cast<const uint4*>(stage + row * C::kStageRow + x * 16),
                    warp * 32 + row < rows && x * 8 < cols);
            }
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              reinterpret_cast<uint4*>(mine)[i] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
            __syncwarp();
            float* to4 = part + c * 32;
            const uint8_t* from4 = stage + (lane >> 3) * C::kStageRow + (lane & 7) * 16;
            uint4 v[8];  // 4 rows of 128 bytes at a time
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = *reinterpret_cast<const uint4*>(from4 + k * 4 * C::kStageRow);
#pragma unroll
            for (int k = 0; k < 8; ++k) st_if(to4 + k * 4 * p.D, v[k], k * 4 < left4 && (lane & 7) * 4 < cols);
          }
        };
        // few rows' parts: a lane's own row goes out as it is, with less code (which is cold) and no way through
        // shared memory
        const bool few = !whole && rows - warp * 32 <= 8 && !__any_sync(0xffffffffu, bad != 0);
        float* own = p.part + (slot + r) * p.D;
#pragma unroll 1
        for (int c = 0; c < DP / 32; ++c) {
          uint32_t o[32];
          tmem_ld32(tmem + c * 32 + lanes, o);
          tmem_wait_ld(o);
          if (few) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              st_if(own + c * 32 + i * 4, make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]),
                    live && c * 32 + i * 4 < p.D);
          } else {
            emit(c, o);
          }
        }
        if (live && !whole) reinterpret_cast<float2*>(p.ml)[slot + r] = make_float2(m, l);
      }
      tc_fence_before();
      asm volatile("bar.sync 2, 128;" ::: "memory");  // before the next segment's q and `bad`
      if (tid == 0) ms.bad = 0;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 5) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)C::kTmem) : "memory");
  }
}

// Joins a row's parts: o = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s. WARPS = 1:
// a warp per row, for many rows; 8: a CTA per row, whose threads share the parts
// (4 ways at D = 256) over the 16-byte words of the row, so that few rows of many
// parts take few round trips to memory. The first parts are loaded before the weights
// are known (16 nodes x 24 heads of 37 parts: 19.3 -> 16.4 us with the kernel above).
constexpr int kJoinThreads = 256, kMaxParts = 1024 + 32;
template <typename T, int WARPS, typename W>
__global__ void __launch_bounds__(kJoinThreads) attn_join_kernel(const __grid_constant__ typename W::Params p) {
  __shared__ float weight[WARPS == 1 ? 1 : kMaxParts];
  __shared__ float4 sum[WARPS == 1 ? 1 : kJoinThreads];
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31;
  const int at_row = WARPS == 1 ? blockIdx.x * (kJoinThreads / 32) + (tid >> 5) : blockIdx.x;
  if (at_row >= p.B * p.n * p.H) return;
  const int head = at_row % p.H, node = at_row / p.H % p.n, b = at_row / p.H / p.n;
  const Seq seq(p, b);
  if (node >= seq.count) return;
  const typename W::Parts at(p, seq, b, node, head);
  const int parts = at.n;
  if (parts == 0) return;  // written whole
  const float2* ml = reinterpret_cast<const float2*>(p.ml);
  T* out = static_cast<T*>(p.o) + b * p.o_batch + node * p.o_node + head * p.o_head;
  // the first parts are on their way while the weights are worked out
  const int words = p.D / 4;
  constexpr int kEarly = WARPS == 1 ? 3 : 8;
  const int ways = WARPS == 1 ? 1 : kJoinThreads / words, way = WARPS == 1 ? 0 : tid / words, w0 = WARPS == 1 ? lane : tid % words;
  constexpr int kPer = WARPS == 1 ? 2 : 1;  // 16-byte words of a row per thread
  float4 early[kEarly][kPer];
#pragma unroll
  for (int k = 0; k < kEarly; ++k) {
    const int s = way + k * ways;
#pragma unroll
    for (int x = 0; x < kPer; ++x)
      early[k][x] = way < ways && s < parts && w0 + 32 * x < words
                        ? *reinterpret_cast<const float4*>(p.part + at(s) * p.D + (w0 + 32 * x) * 4)
                        : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  const float2 own = lane < parts ? ml[at(lane)] : make_float2(-INFINITY, 0.f);
  float M = own.x;  // every warp for itself
  for (int s = lane + 32; s < parts; s += 32) M = fmaxf(M, ml[at(s)].x);
#pragma unroll
  for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  const float wown = ex2(own.x - M);
  float L = lane < parts ? own.y * wown : 0.f;
  if constexpr (WARPS > 1)
    if (tid < 32 && lane < parts) weight[lane] = wown;
  for (int s = lane + 32; s < parts; s += 32) {
    const float2 x = ml[at(s)];
    const float f = ex2(x.x - M);
    L = fmaf(x.y, f, L);
    if constexpr (WARPS > 1)
      if (tid < 32) weight[s] = f;
  }
  L = warp_sum(L);
  auto add = [](float4& a, float f, const float4& v) {
    a.x = fmaf(v.x, f, a.x);
    a.y = fmaf(v.y, f, a.y);
    a.z = fmaf(v.z, f, a.z);
    a.w = fmaf(v.w, f, a.w);
  };
  auto store = [&](int w, const float4& a) {
    const float inv = 1.0f / L;
    *reinterpret_cast<uint2*>(out + w * 4) = make_uint2(pack2<T>(a.x * inv, a.y * inv), pack2<T>(a.z * inv, a.w * inv));
  };
  if constexpr (WARPS == 1) {
    float4 a[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
#pragma unroll
    for (int k = 0; k < kEarly; ++k) {
      const float f = __shfl_sync(0xffffffffu, wown, k);
      if (k < parts) add(a[0], f, early[k][0]), add(a[1], f, early[k][1]);
    }
#pragma unroll 4
    for (int s = kEarly; s < parts; ++s) {
      const float f = s < 32 ? __shfl_sync(0xffffffffu, wown, s & 31) : ex2(ml[at(s)].x - M);
      const float4* v = reinterpret_cast<const float4*>(p.part + at(s) * p.D);
      if (lane < words) add(a[0], f, v[lane]);
      if (lane + 32 < words) add(a[1], f, v[lane + 32]);
    }
    if (lane < words) store(lane, a[0]);
    if (lane + 32 < words) store(lane + 32, a[1]);
  } else {
    __syncthreads();
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    if (way < ways) {
#pragma unroll
      for (int k = 0; k < kEarly; ++k)
        if (way + k * ways < parts) add(a, weight[way + k * ways], early[k][0]);
#pragma unroll 8
      for (int s = way + kEarly * ways; s < parts; s += ways)
        add(a, weight[s], *reinterpret_cast<const float4*>(p.part + at(s) * p.D + w0 * 4));
    }
    sum[tid] = a;
    __syncthreads();
    if (tid < words) {
      for (int k = 1; k < ways; ++k) add(a, 1.0f, sum[k * words + tid]);
      store(tid, a);
    }
  }
}

// ------------------------------------------------------------------ host side
bool tree_sizes_ok(int B, int n, int H, int HK, int D, int n_ctx) {
  return B >= 0 && B <= 65535 && n >= 1 && n <= BTF_TREE_MAX_NODES && HK >= 1 && H >= HK && H % HK == 0 &&
         H <= 65535 && D >= 8 && D <= 256 && D % 8 == 0 && n_ctx >= n && n_ctx <= (1 << 30);
}

int attn_args_ok(const btf_tree_attn* a, const char* what) {
  if (!a) return fail(BTF_ERR_ARG, "%s: null arguments", what);
  if (!tree_sizes_ok(a->B, a->n, a->H, a->HK, a->D, a->n_ctx))
    return fail(BTF_ERR_ARG,
                "%s: need 1 <= n <= %d, H %% HK == 0, D %% 8 == 0 in 8..256 and n_ctx >= n (B %d, n %d, "
                "H %d, HK %d, D %d, n_ctx %d)",
                what, BTF_TREE_MAX_NODES, a->B, a->n, a->H, a->HK, a->D, a->n_ctx);
  if (a->type != BTF_F16 && a->type != BTF_BF16)
    return fail(BTF_ERR_ARG, "%s: q, k, v and o are fp16 or bf16", what);
  if (a->B == 0) return BTF_OK;
  if (!a->q || !a->k || !a->v || !a->o || !a->lens || !a->parents)
    return fail(BTF_ERR_ARG, "%s: null pointer", what);
  auto al = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  if (!al(a->q) || !al(a->k) || !al(a->v) || !al(a->o))
    return fail(BTF_ERR_ARG, "%s: q, k, v and o must be 16-byte aligned", what);
  for (int64_t s : {a->q_batch, a->q_node, a->q_head, a->kv_batch, a->kv_row, a->kv_head, a->o_batch, a->o_node,
                    a->o_head})
    if (s < 0 || s % 8) return fail(BTF_ERR_ARG, "%s: strides must be multiples of 8 elements, >= 0", what);
  if ((a->B > 1 && a->o_batch == 0) || (a->n > 1 && a->o_node == 0) || (a->H > 1 && a->o_head == 0))
    return fail(BTF_ERR_ARG, "%s: the rows of o need strides", what);
  if (a->n_ctx > 1 && a->kv_row == 0) return fail(BTF_ERR_ARG, "%s: the rows of k and v need a stride", what);
  if (!std::isfinite(a->scale)) return fail(BTF_ERR_ARG, "%s: scale must be finite", what);
  if (!a->work || reinterpret_cast<uintptr_t>(a->work) % 256 || a->work_bytes < 256)
    return fail(BTF_ERR_ARG, "%s: workspace null, not 256-byte aligned or too small", what);
  return BTF_OK;
}
bool attn_too_many(const btf_tree_attn& a) {
  return (int64_t)a.B * a.n * a.H > INT32_MAX || (int64_t)a.B * a.HK * ((a.n_ctx + kTile - 1) / kTile) > INT32_MAX / 2;
}

// A map of [batch][rows][heads][D]; a dim with one entry takes any stride.
int encode_rows(CUtensorMap* m, int type, const void* base, int D, int64_t rows, int64_t heads, int64_t batch, int64_t row,
                int64_t head, int64_t batch_stride, const char* what) {
  const EncodeFn fn = encode_fn();
  if (!fn) return fail(BTF_ERR_CUDA, "%s: cuTensorMapEncodeTiled is not available", what);
  const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)rows, (cuuint64_t)heads, (cuuint64_t)batch};
  const cuuint64_t strides[3] = {(cuuint64_t)(rows > 1 ? row * 2 : 16), (cuuint64_t)(heads > 1 ? head * 2 : 16),
                                 (cuuint64_t)(batch > 1 ? batch_stride * 2 : 16)};
  const cuuint32_t box[4] = {64, kTile, 1, 1}, one[4] = {1, 1, 1, 1};
  const CUresult r = fn(m, type == BTF_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                        const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? BTF_OK : fail(BTF_ERR_ARG, "%s: the strides of k and v make no tensor map (%d)", what, (int)r);
}
// The maps of k and v.
int encode_own(CUtensorMap* m, const btf_tree_attn& a, const char* what) {
  const int64_t heads = a.kv_head == 0 ? 1 : a.HK, batch = a.kv_batch == 0 ? 1 : a.B;
  if (int rc = encode_rows(m, a.type, a.k, a.D, a.n_ctx, heads, batch, a.kv_row, a.kv_head, a.kv_batch, what)) return rc;
  return encode_rows(m + 1, a.type, a.v, a.D, a.n_ctx, heads, batch, a.kv_row, a.kv_head, a.kv_batch, what);
}

}  // namespace
}  // namespace btf
