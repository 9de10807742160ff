// Attention for a tree of drafted tokens over a cache (btf_tree_attention), on
// the tcgen05 tensor cores.
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

struct TreeParams {
  const void *q, *v;
  void* o;
  int64_t q_batch, q_node, q_head, kv_batch, kv_row, kv_head, o_batch, o_node, o_head;
  int B, n, H, HK, D, n_ctx, mtiles, ranges;
  int b_mul, h_mul;  // 0: every sequence / kv-head has the same K and V
  const int32_t *lens, *parents, *counts;
  float scale2;     // |scale| log2(e), at least 2^-100 (0 times the -inf of a masked score would be NaN)
  uint32_t q_flip;  // sign bits of two q when scale < 0
  int32_t* first;   // workspace: each sequence's first range, or first tile in the line of all tiles; then tiles per
                    // range, and which of the two it is
  float* part;      // parts: [mtiles][2 ranges][128][D]
  float* ml;        // their (m, l): [mtiles][2 ranges][128][2]
  int* err;
};

// A sequence's nodes, cached rows and tiles.
struct Seq {
  int count, len, tiles;
  Seq() = default;
  __device__ __forceinline__ Seq(const TreeParams& p, int b) {
    count = p.counts ? min(max(p.counts[b], 0), p.n) : p.n;
    len = max(0, min(p.lens[b], p.n_ctx - count));
    tiles = count ? (len + count + kTile - 1) / kTile : 0;
  }
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
struct Segments {
  const TreeParams& p;
  int b, kvh, tile, nt, index;  // the present one; index: in the CTA
  int left;                     // tiles behind it
  Seq seq;
  // Warp-uniform; every warp works it out for itself. Writes the workspace's table when `table`.
  __device__ __forceinline__ Segments(const TreeParams& p_, int range, bool table)
      : p(p_), b(0), kvh(0), tile(0), nt(0), index(0), left(0) {
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
    if (p.B <= 32 && pairs <= p.ranges) {
      const int longest = __reduce_max_sync(0xffffffffu, mine.tiles);
      int per = 1;
      if (__all_sync(0xffffffffu, mine.tiles == 0 || mine.tiles == longest)) {  // (all of one length: no search)
        const int each = p.ranges / max(pairs, 1);
        per = max(1, (longest + each - 1) / each);
      } else {
        const int total = p.HK * __reduce_add_sync(0xffffffffu, mine.tiles);
        per = max(1, (total + p.ranges - 1) / p.ranges);
        // sum ceil(tiles / per) <= total / per + pairs
        int most = pairs < p.ranges ? max(per, (total + p.ranges - pairs - 1) / (p.ranges - pairs)) : max(1, total);
        while (per < most) {
          const int mid = (per + most) / 2;
          if (p.HK * __reduce_add_sync(0xffffffffu, (mine.tiles + mid - 1) / mid) <= p.ranges) most = mid;
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
    int total = 0, t = 0;
    for (int b0 = 0; b0 < p.B; b0 += 32) {
      load(b0);
      t = up_to(mine.tiles * p.HK);
      if (table && b0 + lane < p.B) p.first[b0 + lane] = total + t - mine.tiles * p.HK;
      total += __shfl_sync(0xffffffffu, t, 31);
    }
    const int per = max(1, (total + p.ranges - 1) / p.ranges);
    if (table && lane == 0) p.first[p.B] = per, p.first[p.B + 1] = 0;
    if ((int64_t)range * per >= total) return;
    int start = range * per;
    left = min(per, total - start);
    for (int b0 = 0;; b0 += 32) {  // the sequence that the range starts in
      load(b0);
      t = up_to(mine.tiles * p.HK);
      if (pick(b0, t, &start)) break;
      start -= __shfl_sync(0xffffffffu, t, 31);
    }
    kvh = start / seq.tiles;
    tile = start % seq.tiles;
    nt = min(left, seq.tiles - tile);
    left -= nt;
  }
  __device__ __forceinline__ bool any() const { return nt > 0; }
  __device__ __forceinline__ void next() {
    nt = 0;
    if (left == 0) return;
    if (++kvh == p.HK) {
      kvh = 0;
      do seq = Seq(p, ++b);
      while (seq.tiles == 0);
    }
    ++index;
    tile = 0;
    nt = min(left, seq.tiles);
    left -= nt;
  }
  __device__ __forceinline__ int rows(int mt) const { return min(kRowsM, seq.count * (p.H / p.HK) - mt * kRowsM); }
  __device__ __forceinline__ bool whole() const { return nt == seq.tiles; }
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

// ------------------------------------------------------------------ PTX forms
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w,
                                            uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
      : "memory");
}
// D (fp32) (+)= A (shared memory) x B
__device__ __forceinline__ void mma_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(0u)
      : "memory");
}
// D (fp32) (+)= A (tensor memory) x B
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(0u)
      : "memory");
}
// MN-major, 128-byte swizzle: 64 columns (128 B) x 8 rows (k) per atom; LBO: from
// one 64-column block to the next, SBO: from one group of 8 k to the next.
__device__ __forceinline__ uint64_t smem_desc_mn_sw128(uint32_t addr, uint32_t block_bytes) {
  return (uint64_t)((addr >> 4) & 0x3fffu) | ((uint64_t)(block_bytes >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1u << 46) | ((uint64_t)2u << 61);
}
// kind::f16, D fp32: A and B bf16 or fp16, A K-major; B K-major, or MN-major
__host__ __device__ constexpr uint32_t idesc_f16(bool bf16, bool b_mn, int m, int n) {
  return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((b_mn ? 1u : 0u) << 16) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// 32 lanes x 32 columns of tensor memory; a load's registers are valid after
// tmem_wait_ld on the same array
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
        "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
        "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]),
                 "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]),
                 "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]),
                 "+r"(v[23]), "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]),
                 "+r"(v[30]), "+r"(v[31])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
      "%14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::"r"(v[0]),
      "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
      "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]),
      "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]),
      "r"(v[29]), "r"(v[30]), "r"(v[31]), "r"(addr)
      : "memory");
}
__device__ __forceinline__ void st_if(void* to, uint4 v, bool on) {  // predicated: no branch per store
  asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %5, 0;\n @p st.global.v4.u32 [%0], {%1, %2, %3, %4};\n}\n" ::"l"(to),
               "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w), "r"((int)on)
               : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
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
// One lane of a converged warp. What it guards is issued by one thread with the
// warp's own values (descriptors in uniform registers); behind `lane == 0` each MMA
// costs the warp about 70 cycles to issue, more than a 128 x 64 x 16 one runs.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.b32 %0, 1, 0, p;\n}\n" : "=r"(p)::"memory");
  return p != 0;
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* m) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(m)) : "memory");
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

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, Cfg<DP>::kPerSm)
    tree_attn_kernel(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
                     const __grid_constant__ TreeParams p) {
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
    prefetch_map(&mk);
    prefetch_map(&mv);
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
  const int mt = blockIdx.x % p.mtiles, range = blockIdx.x / p.mtiles, G = p.H / p.HK;
  Segments sg(p, range, blockIdx.x == 0 && warp == 0);
  if (warp == 4) {
    // ---------------------------------------------------------- K and V tiles
    if (lane == 0) {
      int i = 0;
      bool ok = true;
      for (; ok && sg.any(); sg.next()) {
        if (sg.rows(mt) <= 0) continue;
        const int zb = sg.b * p.b_mul, zh = sg.kvh * p.h_mul;
        auto load = [&](const CUtensorMap* map, int j) -> bool {
          const int s = i % C::kStages;
          if (i >= C::kStages && !wait(ms.empty[s], (uint32_t)((i / C::kStages - 1) & 1))) return false;
          const uint32_t bar = smem_u32(&ms.full[s]), dst = sbase + C::kOffRing + s * C::kStage;
          mbar_expect_tx(bar, C::kStage);
#pragma unroll
          for (int c = 0; c < C::kBlocks; ++c)
            tma_load_4d(dst + c * kTile * 128, map, c * 64, (sg.tile + j) * kTile, zh, zb, bar);
          ++i;
          return true;
        };
        for (int j = -kAhead; ok && j < sg.nt; ++j) {
          if (j + kAhead < sg.nt) ok = load(&mk, j + kAhead);
          if (ok && j >= 0) ok = load(&mv, j);
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
      if (sg.rows(mt) <= 0) continue;
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
      const int rows = sg.rows(mt);
      if (rows <= 0) continue;
      const int active = (rows + 31) >> 5;  // warps with rows; the others only keep step
      const Seq& seq = sg.seq;
      const int r = tid, rr = mt * kRowsM + r;
      const bool live = r < rows;
      const int node = live ? rr / G : 0, head = sg.kvh * G + (live ? rr % G : 0);
      // the warp's q rows: 4 rows of 128 bytes at a time, 8 lanes each
      if (warp < active) {
        const T* q = static_cast<const T*>(p.q) + sg.b * p.q_batch;
        const int64_t qo = live ? node * p.q_node + head * p.q_head : -1;
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
      if (warp < active) {
        uint64_t mm[2];
        tree_masks(p.parents + (int64_t)sg.b * p.n, seq.count, mm);
        const uint64_t m0 = __shfl_sync(0xffffffffu, mm[0], node & 31), m1 = __shfl_sync(0xffffffffu, mm[1], node & 31);
        if (live) mask = node < 32 ? m0 : m1;
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
        const int64_t slot = (int64_t)mt * 2 * p.ranges + 2 * range + (sg.index > 0);
        const uint64_t bad = ms.bad & mask;
        // where this lane's row goes (the lanes ask each other), or the first of its words of the parts
        const int64_t to = sg.b * p.o_batch + node * p.o_node + head * p.o_head;
        float* part = p.part + (slot * kRowsM + warp * 32 + (lane >> 3)) * p.D + (lane & 7) * 4;
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
        float* own = p.part + (slot * kRowsM + r) * p.D;
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
        if (live && !whole) reinterpret_cast<float2*>(p.ml)[slot * kRowsM + r] = make_float2(m, l);
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
constexpr int kJoinThreads = 256, kMaxParts = 1024;
template <typename T, int WARPS>
__global__ void __launch_bounds__(kJoinThreads) tree_join_kernel(const __grid_constant__ TreeParams p) {
  __shared__ float weight[WARPS == 1 ? 1 : kMaxParts];
  __shared__ float4 sum[WARPS == 1 ? 1 : kJoinThreads];
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, G = p.H / p.HK;
  const int at_row = WARPS == 1 ? blockIdx.x * (kJoinThreads / 32) + (tid >> 5) : blockIdx.x;
  if (at_row >= p.B * p.n * p.H) return;
  const int head = at_row % p.H, node = at_row / p.H % p.n, b = at_row / p.H / p.n;
  const int per = p.first[p.B], first = p.first[b];
  const Seq seq(p, b);
  if (node >= seq.count) return;
  int r0, parts;
  bool second = false;  // whether r0 begins with another pair's tiles
  if (p.first[p.B + 1]) {
    parts = (seq.tiles + per - 1) / per;
    r0 = first + head / G * parts;
  } else {
    const int t0 = first + head / G * seq.tiles, t1 = t0 + seq.tiles - 1;
    r0 = t0 / per, parts = t1 / per - r0 + 1;
    second = r0 * per < t0;
  }
  if (parts == 1) return;  // written whole
  const int rr = node * G + head % G;
  const int64_t base = ((int64_t)(rr / kRowsM) * 2 * p.ranges + 2 * r0) * kRowsM + rr % kRowsM;
  auto at = [&](int s) { return base + (2 * s + (s == 0 && second)) * kRowsM; };
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

bool tree_sizes_ok(int B, int n, int H, int HK, int D, int n_ctx) {
  return B >= 0 && B <= 65535 && n >= 1 && n <= BTF_TREE_MAX_NODES && HK >= 1 && H >= HK && H % HK == 0 &&
         H <= 65535 && D >= 8 && D <= 256 && D % 8 == 0 && n_ctx >= n && n_ctx <= (1 << 30);
}

// The launch's shape and its workspace: the table of first tiles, then the parts
// (two per range and M tile) and their (m, l).
struct Plan {
  int mtiles, ranges;
  int64_t off_part, off_ml, bytes;
};
Plan tree_plan(const DeviceInfo& d, int B, int n, int H, int HK, int D, int n_ctx) {
  Plan r;
  r.mtiles = (n * (H / HK) + kRowsM - 1) / kRowsM;
  const int64_t tiles = (int64_t)B * HK * ((n_ctx + kTile - 1) / kTile);
  const int64_t slots = std::max(1, d.sm_count * (D <= 128 ? 2 : 1) / r.mtiles);
  r.ranges = (int)std::max<int64_t>(1, std::min(slots, tiles));
  r.off_part = ((int64_t)(B + 2) * 4 + 255) / 256 * 256;
  const int64_t rows = (int64_t)r.mtiles * 2 * r.ranges * kRowsM;
  r.off_ml = r.off_part + rows * D * 4;
  r.bytes = r.off_ml + rows * 8;
  return r;
}

int encode_kv(CUtensorMap* m, const btf_tree_attn& a, const void* base, bool b_one, bool h_one) {
  const EncodeFn fn = encode_fn();
  if (!fn) return fail(BTF_ERR_CUDA, "btf_tree_attention: cuTensorMapEncodeTiled is not available");
  const cuuint64_t dims[4] = {(cuuint64_t)a.D, (cuuint64_t)a.n_ctx, (cuuint64_t)(h_one ? 1 : a.HK),
                              (cuuint64_t)(b_one ? 1 : a.B)};
  // a dim with one entry takes any stride
  const cuuint64_t strides[3] = {(cuuint64_t)(a.n_ctx > 1 ? a.kv_row * 2 : 16), (cuuint64_t)(h_one ? 16 : a.kv_head * 2),
                                 (cuuint64_t)(b_one ? 16 : a.kv_batch * 2)};
  const cuuint32_t box[4] = {64, kTile, 1, 1}, one[4] = {1, 1, 1, 1};
  const CUresult r = fn(m, a.type == BTF_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                        const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? BTF_OK
                           : fail(BTF_ERR_ARG, "btf_tree_attention: the strides of k and v make no tensor map (%d)", (int)r);
}

template <typename T, int DP>
cudaError_t launch_tree(const CUtensorMap& mk, const CUtensorMap& mv, const TreeParams& p, cudaStream_t st) {
  return launch_pdl(tree_attn_kernel<T, DP>, dim3((unsigned)(p.ranges * p.mtiles)), dim3(kThreads), (size_t)Cfg<DP>::kSmem, st, mk,
                    mv, p);
}
template <typename T>
cudaError_t launch_tree_d(const CUtensorMap& mk, const CUtensorMap& mv, const TreeParams& p, int sms, cudaStream_t st) {
  const cudaError_t e = p.D <= 64    ? launch_tree<T, 64>(mk, mv, p, st)
                        : p.D <= 128 ? launch_tree<T, 128>(mk, mv, p, st)
                        : p.D <= 192 ? launch_tree<T, 192>(mk, mv, p, st)
                                     : launch_tree<T, 256>(mk, mv, p, st);
  if (e != cudaSuccess || p.ranges == 1) return e;
  const int64_t rows = (int64_t)p.B * p.n * p.H;  // at most INT32_MAX
  // a CTA per row while all of them are resident at once
  if (rows <= 8 * sms) return launch_pdl(tree_join_kernel<T, 8>, dim3((unsigned)rows), dim3(kJoinThreads), 0, st, p);
  return launch_pdl(tree_join_kernel<T, 1>, dim3((unsigned)((rows + 7) / 8)), dim3(kJoinThreads), 0, st, p);
}

// The join runs between two launches that take all of shared memory: it asks for
// the same split of the SM's storage, which changes only on an idle SM.
template <typename T, int WARPS>
cudaError_t join_carveout() {
  return cudaFuncSetAttribute(tree_join_kernel<T, WARPS>, cudaFuncAttributePreferredSharedMemoryCarveout,
                              cudaSharedmemCarveoutMaxShared);
}
template <typename T, int DP>
cudaError_t allow_smem(const DeviceInfo& d) {
  static_assert(Cfg<DP>::kSmem * Cfg<DP>::kPerSm <= 228 * 1024 - 1024 * Cfg<DP>::kPerSm);
  if (Cfg<DP>::kSmem > d.optin_smem) return cudaErrorInvalidValue;
  return cudaFuncSetAttribute(tree_attn_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<DP>::kSmem);
}

}  // namespace

int tree_attn_setup(DeviceInfo& d) {
  for (cudaError_t e : {allow_smem<__half, 64>(d), allow_smem<__half, 128>(d), allow_smem<__half, 192>(d),
                        allow_smem<__half, 256>(d), allow_smem<__nv_bfloat16, 64>(d), allow_smem<__nv_bfloat16, 128>(d),
                        allow_smem<__nv_bfloat16, 192>(d), allow_smem<__nv_bfloat16, 256>(d),
                        join_carveout<__half, 1>(), join_carveout<__half, 8>(), join_carveout<__nv_bfloat16, 1>(),
                        join_carveout<__nv_bfloat16, 8>()})
    if (e != cudaSuccess) return cuda_fail(e, "tree_attn_kernel attributes");
  return BTF_OK;
}

}  // namespace btf

using namespace btf;

extern "C" {

int64_t btf_tree_attention_work(int B, int n, int H, int HK, int D, int n_ctx) {
  if (!tree_sizes_ok(B, n, H, HK, D, n_ctx)) {
    fail(BTF_ERR_ARG, "btf_tree_attention_work: bad sizes (B %d, n %d, H %d, HK %d, D %d, n_ctx %d)", B, n, H, HK, D,
         n_ctx);
    return -1;
  }
  const DeviceInfo* dev = current_device();
  if (!dev) return -1;
  return tree_plan(*dev, B, n, H, HK, D, n_ctx).bytes;
}

int btf_tree_attention(const btf_tree_attn* a, void* stream) {
  if (!a) return fail(BTF_ERR_ARG, "btf_tree_attention: null arguments");
  if (!tree_sizes_ok(a->B, a->n, a->H, a->HK, a->D, a->n_ctx))
    return fail(BTF_ERR_ARG,
                "btf_tree_attention: need 1 <= n <= %d, H %% HK == 0, D %% 8 == 0 in 8..256 and n_ctx >= n (B %d, n %d, "
                "H %d, HK %d, D %d, n_ctx %d)",
                BTF_TREE_MAX_NODES, a->B, a->n, a->H, a->HK, a->D, a->n_ctx);
  if (a->type != BTF_F16 && a->type != BTF_BF16)
    return fail(BTF_ERR_ARG, "btf_tree_attention: q, k, v and o are fp16 or bf16");
  if (a->B == 0) return BTF_OK;
  if (!a->q || !a->k || !a->v || !a->o || !a->lens || !a->parents)
    return fail(BTF_ERR_ARG, "btf_tree_attention: null pointer");
  auto al = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  if (!al(a->q) || !al(a->k) || !al(a->v) || !al(a->o))
    return fail(BTF_ERR_ARG, "btf_tree_attention: q, k, v and o must be 16-byte aligned");
  for (int64_t s : {a->q_batch, a->q_node, a->q_head, a->kv_batch, a->kv_row, a->kv_head, a->o_batch, a->o_node,
                    a->o_head})
    if (s < 0 || s % 8) return fail(BTF_ERR_ARG, "btf_tree_attention: strides must be multiples of 8 elements, >= 0");
  if ((a->B > 1 && a->o_batch == 0) || (a->n > 1 && a->o_node == 0) || (a->H > 1 && a->o_head == 0))
    return fail(BTF_ERR_ARG, "btf_tree_attention: the rows of o need strides");
  if (a->n_ctx > 1 && a->kv_row == 0) return fail(BTF_ERR_ARG, "btf_tree_attention: the rows of k and v need a stride");
  if (!std::isfinite(a->scale)) return fail(BTF_ERR_ARG, "btf_tree_attention: scale must be finite");
  if (!a->work || reinterpret_cast<uintptr_t>(a->work) % 256 || a->work_bytes < 256)
    return fail(BTF_ERR_ARG, "btf_tree_attention: workspace null, not 256-byte aligned or too small");
  const DeviceInfo* dev = current_device();
  if (!dev) return BTF_ERR_STATE;
  const Plan plan = tree_plan(*dev, a->B, a->n, a->H, a->HK, a->D, a->n_ctx);
  if (a->work_bytes < plan.bytes)
    return fail(BTF_ERR_ARG, "btf_tree_attention: the workspace has %lld bytes, %lld are needed", (long long)a->work_bytes,
                (long long)plan.bytes);
  if (plan.ranges > kMaxParts || (int64_t)a->B * a->n * a->H > INT32_MAX ||
      (int64_t)a->B * a->HK * ((a->n_ctx + kTile - 1) / kTile) > INT32_MAX / 2)
    return fail(BTF_ERR_UNSUPPORTED, "btf_tree_attention: too many sequences and heads for one launch");
  const bool b_one = a->B == 1 || a->kv_batch == 0, h_one = a->HK == 1 || a->kv_head == 0;
  CUtensorMap mk, mv;
  if (int rc = encode_kv(&mk, *a, a->k, b_one, h_one)) return rc;
  if (int rc = encode_kv(&mv, *a, a->v, b_one, h_one)) return rc;
  uint8_t* work = static_cast<uint8_t*>(a->work);
  const TreeParams p{a->q, a->v, a->o, a->q_batch, a->q_node, a->q_head, a->kv_batch, a->kv_row, a->kv_head, a->o_batch,
                     a->o_node, a->o_head, a->B, a->n, a->H, a->HK, a->D, a->n_ctx, plan.mtiles, plan.ranges,
                     b_one ? 0 : 1, h_one ? 0 : 1, a->lens, a->parents, a->counts,
                     std::max(std::fabs(a->scale) * 1.4426950408889634f, 0x1p-100f), a->scale < 0 ? 0x80008000u : 0u,
                     reinterpret_cast<int32_t*>(work), reinterpret_cast<float*>(work + plan.off_part),
                     reinterpret_cast<float*>(work + plan.off_ml), dev->err_word};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e =
      a->type == BTF_F16 ? launch_tree_d<__half>(mk, mv, p, dev->sm_count, st)
                              : launch_tree_d<__nv_bfloat16>(mk, mv, p, dev->sm_count, st);
  return e == cudaSuccess ? BTF_OK : cuda_fail(e, "btf_tree_attention");
}

}  // extern "C"
