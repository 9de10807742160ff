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
// One CTA: a range of 64-row tiles of the cache for one (sequence, kv-head, M
// tile). Warp 4 loads K and V tiles by TMA into a ring, warp 5 issues the MMAs,
// warps 0..3 hold one q row per thread:
//   S = Q K^T (64 columns of tensor memory, two of them in turn) -> registers,
//   mask, running maximum, p = 2^(s - m) -> 16 bits, back into the tensor memory of
//   S, from where it is the A operand of O += P V (V as it lies: MN-major B).
// S of the next tile is computed during the softmax of this one. The maximum that p
// is taken against only moves when a row's grows by more than 2^8 (m then jumps and
// O is rescaled in tensor memory); p stays below 2^8, which the type holds, and
// the sum below it is exact in fp32 all the same.
//
// p is rounded to the type of V (the MMA takes one type): eps / 2 per term, as much
// as the output's own rounding at most. fp16 p carry a factor 2^7, so that those
// down to 2^-32 of the largest still count. Scores, maxima, sums and O are fp32.
//
// The cache is split over CTAs where there are fewer (sequence, kv-head, M tile)
// than SMs; the parts are joined by a second kernel.
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
constexpr int kMaxSplits = 256;
constexpr uint64_t kWaitNs = 1000000000ull;
constexpr float kLag = 8.0f;  // log2 of how far a row's maximum may run ahead of m

template <int DP>  // D padded to whole 128-byte swizzle rows
struct Cfg {
  static constexpr int kBlocks = DP / 64;          // 64-column blocks
  static constexpr int kQBytes = kRowsM * DP * 2;  // [block][128 rows][128 B], SW128
  static constexpr int kStage = kTile * DP * 2;    // [block][64 rows][128 B], SW128
  // one CTA per SM at 192 and 256 (Q alone takes 48 and 64 KB), two below: each
  // has about 64 KB of copies in flight, which one SM's share of the memory rate needs
  static constexpr int kStages = DP == 256 ? 5 : DP == 192 ? 6 : DP == 128 ? 4 : 10;
  static constexpr int kTmem = DP <= 128 ? 256 : 512;  // O: DP columns; S (P): 2 x 64
  static constexpr int kPerSm = DP <= 128 ? 2 : 1;
  static constexpr int kOffRing = kQBytes;
  static constexpr int kOffMisc = kOffRing + kStages * kStage;
  static constexpr int kSmem = 1024 + kOffMisc + 1280;
};

struct TreeParams {
  const void *q, *v;
  void* o;
  int64_t q_batch, q_node, q_head, kv_batch, kv_row, kv_head, o_batch, o_node, o_head;
  int B, n, H, HK, D, n_ctx, mtiles, splits;
  int b_mul, h_mul;  // 0: every sequence / kv-head has the same K and V
  const int32_t *lens, *parents, *counts;
  float scale2;  // scale * log2(e)
  float* part;   // [splits][B n H][D], then (m, l) [splits][B n H][2]
  int* err;
};

// The sequence's nodes, cached rows and tiles.
struct Seq {
  int count, len, tiles, per;  // tiles of all its rows; tiles per split
  __device__ __forceinline__ Seq(const TreeParams& p, int b) {
    count = p.counts ? min(max(p.counts[b], 0), p.n) : p.n;
    len = max(0, min(p.lens[b], p.n_ctx - count));
    tiles = (len + count + kTile - 1) / kTile;
    per = (tiles + p.splits - 1) / p.splits;
  }
};

// Itself and its ancestors, as bits, for the nodes of a tree: pointer doubling over
// the parents (a parent that is not an earlier node hangs on the cache). One warp.
__device__ __forceinline__ void tree_masks(const int32_t* parents, int n, uint64_t* out, int* jump) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int j = lane + 32 * r, pj = j < n ? parents[j] : -1;
    jump[j] = pj >= 0 && pj < j ? pj : -1;
    out[j] = 1ull << j;
  }
  __syncwarp();
  for (int s = 0; s < 6; ++s) {
    uint64_t m[2];
    int jj[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int j = lane + 32 * r, a = jump[j];
      m[r] = out[j] | (a >= 0 ? out[a] : 0ull);
      jj[r] = a >= 0 ? jump[a] : -1;
    }
    __syncwarp();
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      out[lane + 32 * r] = m[r];
      jump[lane + 32 * r] = jj[r];
    }
    __syncwarp();
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
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float ex2(float x) {  // 2^x, 2 ulp; 0 below 2^-126
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  Pack<T, 2> r;
  r.set(0, a);
  r.set(1, b);
  return r.w[0];
}

// Shared memory behind the ring.
struct Misc {
  uint64_t full[10], empty[10], s_full[2], p_ready[2], pv_done, final;  // mbarriers
  uint64_t masks[64];
  int jump[64];
  unsigned long long bad;  // nodes with an infinity or NaN in V
  uint32_t tmem;
  int abort;
};
static_assert(sizeof(Misc) <= 1280);

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, Cfg<DP>::kPerSm)
    tree_attn_kernel(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
                     const __grid_constant__ TreeParams p) {
  using C = Cfg<DP>;
  constexpr bool kBf16 = std::is_same_v<T, __nv_bfloat16>;
  constexpr float kBias = kBf16 ? 0.0f : 7.0f;  // fp16 p times 2^7 (below 2^8 * 2^7)
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw), sbase = (raw + 1023) & ~1023u;
  uint8_t* smem = smem_raw + (sbase - raw);
  Misc& ms = *reinterpret_cast<Misc*>(smem + C::kOffMisc);
  volatile int* abort_flag = &ms.abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (warp == 5) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ms.tmem)),
                 "r"((uint32_t)C::kTmem)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ms.tmem, tmem_s = tmem + DP;
  pdl_launch_dependents();
  pdl_wait();

  const int mt = blockIdx.x % p.mtiles, sp = blockIdx.x / p.mtiles % p.splits, bh = blockIdx.x / p.mtiles / p.splits;
  const int b = bh / p.HK, kvh = bh % p.HK, G = p.H / p.HK;
  const Seq seq(p, b);
  const int j0 = sp * seq.per, nt = min(seq.per, seq.tiles - j0);  // this CTA's tiles
  const int rows = min(kRowsM, seq.count * G - mt * kRowsM);
  if (nt > 0 && rows > 0) {  // (the same for the whole CTA)
    const int active = (rows + 31) >> 5;  // warps with q rows
    if (tid == 0) {
      for (int i = 0; i < C::kStages; ++i) {
        mbar_init(smem_u32(&ms.full[i]), 1);
        mbar_init(smem_u32(&ms.empty[i]), 1);
      }
      for (int i = 0; i < 2; ++i) {
        mbar_init(smem_u32(&ms.s_full[i]), 1);
        mbar_init(smem_u32(&ms.p_ready[i]), active);
      }
      mbar_init(smem_u32(&ms.pv_done), 1);
      mbar_init(smem_u32(&ms.final), 1);
      ms.bad = 0;
      ms.abort = 0;
      fence_mbar_init();
    }
    __syncthreads();
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
    int issued = 0;  // warp 4: ring loads issued
    if (warp == 4) {
      // -------------------------------------------------------- K and V tiles
      if (lane == 0) {
        const int zb = b * p.b_mul, zh = kvh * p.h_mul;
        for (int i = 0; i < 2 * nt; ++i) {  // K of tile 0, V of tile 0, K of tile 1, ...
          const int s = i % C::kStages;
          if (i >= C::kStages && !wait(ms.empty[s], (uint32_t)((i / C::kStages - 1) & 1))) break;
          const uint32_t bar = smem_u32(&ms.full[s]), dst = sbase + C::kOffRing + s * C::kStage;
          mbar_expect_tx(bar, C::kStage);
#pragma unroll
          for (int c = 0; c < C::kBlocks; ++c)
            tma_load_4d(dst + c * kTile * 128, i & 1 ? &mv : &mk, c * 64, (j0 + (i >> 1)) * kTile, zh, zb, bar);
          issued = i + 1;
        }
      }
    } else {
      // the q rows, and the trees' masks (warp 0)
      if (warp == 0) tree_masks(p.parents + (int64_t)b * p.n, seq.count, ms.masks, ms.jump);
      const T* q = static_cast<const T*>(p.q) + b * p.q_batch + (int64_t)kvh * G * p.q_head;
      const int t = warp == 5 ? 128 + lane : tid;
      for (int i = t; i < active * 32 * (DP / 8); i += 160) {
        const int r = i / (DP / 8), c = i % (DP / 8);  // row, 16-byte chunk
        uint4 v = make_uint4(0, 0, 0, 0);
        if (r < rows && c * 8 < p.D) {
          const int rr = mt * kRowsM + r;
          v = *reinterpret_cast<const uint4*>(q + (rr / G) * p.q_node + (rr % G) * p.q_head + c * 8);
        }
        *reinterpret_cast<uint4*>(smem + (c >> 3) * (kRowsM * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = v;
      }
      fence_proxy_async_smem();
      asm volatile("bar.sync 1, 160;" ::: "memory");  // warps 0..3 and 5
      if (warp == 5) {
        // ------------------------------------------------------ MMAs
        if (lane == 0) {
          constexpr uint32_t kQk = idesc_f16(kBf16, false, kRowsM, kTile), kPv = idesc_f16(kBf16, true, kRowsM, DP);
          const uint64_t qd = smem_desc_sw128(sbase);
          auto qk = [&](int j) -> bool {  // S of tile j
            const int i = 2 * j, s = i % C::kStages;
            if (!wait(ms.full[s], (uint32_t)((i / C::kStages) & 1))) return false;
            if (j >= 2 && !wait(ms.pv_done, (uint32_t)(j & 1))) return false;  // P of tile j - 2 has been read
            tc_fence_after();
            const uint64_t kd = smem_desc_sw128(sbase + C::kOffRing + s * C::kStage);
#pragma unroll
            for (int c = 0; c < DP / 16; ++c)
              mma_f16_ss(tmem_s + (j & 1) * kTile, qd + (((c >> 2) * kRowsM * 128 + (c & 3) * 32) >> 4),
                         kd + (((c >> 2) * kTile * 128 + (c & 3) * 32) >> 4), kQk, c > 0);
            mma_commit(smem_u32(&ms.s_full[j & 1]));
            mma_commit(smem_u32(&ms.empty[s]));
            return true;
          };
          bool ok = qk(0);
          for (int j = 0; ok && j < nt; ++j) {
            if (j + 1 < nt && !qk(j + 1)) break;
            const int i = 2 * j + 1, s = i % C::kStages;
            if (!wait(ms.full[s], (uint32_t)((i / C::kStages) & 1))) break;
            if (!wait(ms.p_ready[j & 1], (uint32_t)((j >> 1) & 1))) break;
            tc_fence_after();
            const uint64_t vd = smem_desc_mn_sw128(sbase + C::kOffRing + s * C::kStage, kTile * 128);
#pragma unroll
            for (int c = 0; c < kTile / 16; ++c)
              mma_f16_ts(tmem, tmem_s + (j & 1) * kTile + c * 8, vd + (c * 2048 >> 4), kPv, j > 0 || c > 0);
            mma_commit(smem_u32(&ms.empty[s]));
            mma_commit(smem_u32(&ms.pv_done));
          }
          mma_commit(smem_u32(&ms.final));  // completes when every MMA issued above has finished
          mbar_wait_bounded(smem_u32(&ms.final), 0, kWaitNs);
        }
      } else if (warp < active) {
        // ------------------------------------------------------ softmax, one row per thread
        const uint32_t lanes = (uint32_t)(warp * 32) << 16;
        const int r = tid, rr = mt * kRowsM + r;
        const bool live = r < rows;
        const int node = live ? rr / G : 0;
        const uint64_t mask = live ? ms.masks[node] : 0ull;
        float m = -INFINITY, l = 0.f;
        bool ok = true;
        for (int j = 0; j < nt; ++j) {
          const int t0 = (j0 + j) * kTile;
          if (!warp_wait(ms.s_full[j & 1], (uint32_t)((j >> 1) & 1))) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t ts = tmem_s + (j & 1) * kTile + lanes;
          uint32_t s0[32], s1[32];
          tmem_ld32(ts, s0);
          tmem_ld32(ts + 32, s1);
          tmem_wait_ld(s0);
          tmem_wait_ld(s1);
          float mx = -INFINITY;
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            s0[i] = __float_as_uint(__uint_as_float(s0[i]) * p.scale2);
            s1[i] = __float_as_uint(__uint_as_float(s1[i]) * p.scale2);
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
#pragma unroll
          for (int i = 0; i < 32; ++i) mx = fmaxf(mx, fmaxf(__uint_as_float(s0[i]), __uint_as_float(s1[i])));
          if (__any_sync(0xffffffffu, mx > m + kLag)) {
            const float mn = fmaxf(m, mx), f = m == -INFINITY ? (l == 0.f ? 0.f : 1.f) : ex2(m - mn);
            m = mn;
            l *= f;
            if (j > 0) {
              if (!warp_wait(ms.pv_done, (uint32_t)((j - 1) & 1))) {
                ok = false;
                break;
              }
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
          const float sub = (m == -INFINITY ? 0.f : m) - kBias;
          float l0 = 0.f, l1 = 0.f;
          uint32_t pk[32];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float a = ex2(__uint_as_float(s0[2 * i]) - sub), c = ex2(__uint_as_float(s0[2 * i + 1]) - sub);
            const float e = ex2(__uint_as_float(s1[2 * i]) - sub), g = ex2(__uint_as_float(s1[2 * i + 1]) - sub);
            l0 += a + c;
            l1 += e + g;
            pk[i] = pack2<T>(a, c);
            pk[16 + i] = pack2<T>(e, g);
          }
          l += l0 + l1;
          tmem_st32(ts, pk);
          tmem_wait_st();
          if (t0 + kTile > seq.len) {
            // V rows behind the last node would meet p = 0, and so would a node's row for
            // those that do not see it: 0 x NaN. The former are zeroed; of the latter,
            // infinities and NaN are, and added at the end for those that see them.
            const int i = 2 * j + 1, s = i % C::kStages;
            if (!warp_wait(ms.full[s], (uint32_t)((i / C::kStages) & 1))) {
              ok = false;
              break;
            }
            uint8_t* vs = smem + C::kOffRing + s * C::kStage;
            const int first = max(0, seq.len - t0);  // tile rows of nodes and behind
            for (int e = tid; e < (kTile - first) * (DP / 8); e += active * 32) {
              const int row = first + e / (DP / 8), c = e % (DP / 8), nd = t0 + row - seq.len;
              uint4* at = reinterpret_cast<uint4*>(vs + (c >> 3) * (kTile * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4));
              if (nd >= seq.count) {
                *at = make_uint4(0, 0, 0, 0);
                continue;
              }
              uint4 v = *at;
              constexpr uint32_t kExp = kBf16 ? 0x7f80u : 0x7c00u;
              uint32_t w[4] = {v.x, v.y, v.z, v.w};
              bool any = false;
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                if ((w[x] & kExp) == kExp) w[x] &= 0xffff0000u, any = true;
                if (((w[x] >> 16) & kExp) == kExp) w[x] &= 0xffffu, any = true;
              }
              if (any) {
                *at = make_uint4(w[0], w[1], w[2], w[3]);
                atomicOr(&ms.bad, 1ull << nd);
              }
            }
            fence_proxy_async_smem();
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&ms.p_ready[j & 1]));
        }
        // ------------------------------------------------------ the output row, or this split's part of it
        ok = ok && warp_wait(ms.pv_done, (uint32_t)((nt - 1) & 1));
        asm volatile("bar.sync 2, %0;" ::"r"(active * 32) : "memory");  // every warp's part of `bad` is in
        if (ok) {
          tc_fence_after();
          const bool whole = seq.per >= seq.tiles;
          const int head = kvh * G + (live ? rr % G : 0);
          const int64_t row = ((int64_t)b * p.n + node) * p.H + head, all = (int64_t)p.B * p.n * p.H;
          const float inv = whole ? 1.0f / l : 1.0f;
          T* out = static_cast<T*>(p.o) + b * p.o_batch + node * p.o_node + head * p.o_head;
          float* part = p.part + (sp * all + row) * p.D;
          const uint64_t bad = ms.bad & mask;
          const T* v = static_cast<const T*>(p.v) + b * p.kv_batch + kvh * p.kv_head;
#pragma unroll 1
          for (int c = 0; c < DP / 32; ++c) {
            uint32_t o[32];
            tmem_ld32(tmem + c * 32 + lanes, o);
            tmem_wait_ld(o);
            if (!live) continue;
            if (bad) {
              for (uint64_t left = bad; left; left &= left - 1) {
                const T* vr = v + (int64_t)(seq.len + __ffsll((long long)left) - 1) * p.kv_row + c * 32;
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                  const float x = c * 32 + i < p.D ? to_f32(vr[i]) : 0.f;
                  if (!(fabsf(x) < INFINITY)) o[i] = __float_as_uint(__uint_as_float(o[i]) + x);
                }
              }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if (c * 32 + i * 8 >= p.D) break;
              float f[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(o[i * 8 + e]) * inv;
              if (whole) {
                Pack<T, 8> y;
#pragma unroll
                for (int e = 0; e < 8; ++e) y.set(e, f[e]);
                y.store(out + c * 32 + i * 8);
              } else {
                float4* d = reinterpret_cast<float4*>(part + c * 32 + i * 8);
                d[0] = make_float4(f[0], f[1], f[2], f[3]);
                d[1] = make_float4(f[4], f[5], f[6], f[7]);
              }
            }
          }
          if (live && !whole) {
            float* ml = p.part + (int64_t)p.splits * all * p.D + (sp * all + row) * 2;
            ml[0] = m;
            ml[1] = l;
          }
        }
      }
    }
    if (warp == 4 && lane == 0 && *abort_flag) {  // leave no copy in flight into this CTA's shared memory (bounded)
      for (int i = max(0, issued - C::kStages); i < issued; ++i)
        mbar_wait_bounded(smem_u32(&ms.full[i % C::kStages]), (uint32_t)((i / C::kStages) & 1), kWaitNs / 10);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 5) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)C::kTmem) : "memory");
  }
}

// Joins the splits of a row: o = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s. A warp per row.
template <typename T>
__global__ void __launch_bounds__(256) tree_join_kernel(const __grid_constant__ TreeParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t all = (int64_t)p.B * p.n * p.H, row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= all) return;
  const int head = (int)(row % p.H), node = (int)(row / p.H % p.n), b = (int)(row / p.H / p.n);
  const Seq seq(p, b);
  if (node >= seq.count || seq.per >= seq.tiles) return;  // not a node, or already written whole
  const int splits = (seq.tiles + seq.per - 1) / seq.per;
  const float2* ml = reinterpret_cast<const float2*>(p.part + (int64_t)p.splits * all * p.D) + row;
  float M = -INFINITY, L = 0.f;
  for (int s = lane; s < splits; s += 32) M = fmaxf(M, ml[s * all].x);
#pragma unroll
  for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  for (int s = lane; s < splits; s += 32) L += ml[s * all].y * ex2(ml[s * all].x - M);
  L = warp_sum(L);
  T* out = static_cast<T*>(p.o) + b * p.o_batch + node * p.o_node + head * p.o_head;
  for (int c = lane * 4; c < p.D; c += 128) {
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int s = 0; s < splits; ++s) {
      const float f = ex2(ml[s * all].x - M);
      const float4 v = *reinterpret_cast<const float4*>(p.part + (s * all + row) * p.D + c);
      a.x = fmaf(v.x, f, a.x);
      a.y = fmaf(v.y, f, a.y);
      a.z = fmaf(v.z, f, a.z);
      a.w = fmaf(v.w, f, a.w);
    }
    Pack<T, 4> y;
    y.set(0, a.x / L);
    y.set(1, a.y / L);
    y.set(2, a.z / L);
    y.set(3, a.w / L);
    y.store(out + c);
  }
}

bool tree_sizes_ok(int B, int n, int H, int HK, int D, int n_ctx) {
  return B >= 0 && B <= 65535 && n >= 1 && n <= BTF_TREE_MAX_NODES && HK >= 1 && H >= HK && H % HK == 0 &&
         H <= 65535 && D >= 8 && D <= 256 && D % 8 == 0 && n_ctx >= n && n_ctx <= (1 << 30);
}

// Splits of the cache: the count with the least time for a full cache, by the
// number of waves of CTAs and the tiles of each; a CTA's start and end cost about
// kFixed tiles.
int tree_splits(const DeviceInfo& d, int B, int n, int H, int HK, int D, int n_ctx) {
  constexpr int kFixed = 4;
  const int64_t units = (int64_t)B * HK * ((n * (H / HK) + kRowsM - 1) / kRowsM);
  const int64_t slots = (int64_t)d.sm_count * (D <= 128 ? 2 : 1), tiles = (n_ctx + kTile - 1) / kTile;
  int best = 1;
  int64_t least = INT64_MAX;
  for (int s = 1; s <= kMaxSplits && s <= tiles; ++s) {
    const int64_t waves = (units * s + slots - 1) / slots, t = waves * ((tiles + s - 1) / s + kFixed);
    if (t < least) least = t, best = s;
  }
  return best;
}

int64_t work_bytes(int splits, int B, int n, int H, int D) {
  return std::max<int64_t>(256, splits > 1 ? (int64_t)splits * B * n * H * (D + 2) * 4 : 0);
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
  return launch_pdl(tree_attn_kernel<T, DP>, dim3((unsigned)((int64_t)p.B * p.HK * p.splits * p.mtiles)), dim3(kThreads),
                    (size_t)Cfg<DP>::kSmem, st, mk, mv, p);
}
template <typename T>
cudaError_t launch_tree_d(const CUtensorMap& mk, const CUtensorMap& mv, const TreeParams& p, cudaStream_t st) {
  const cudaError_t e = p.D <= 64    ? launch_tree<T, 64>(mk, mv, p, st)
                        : p.D <= 128 ? launch_tree<T, 128>(mk, mv, p, st)
                        : p.D <= 192 ? launch_tree<T, 192>(mk, mv, p, st)
                                     : launch_tree<T, 256>(mk, mv, p, st);
  if (e != cudaSuccess || p.splits == 1) return e;
  return launch_pdl(tree_join_kernel<T>, dim3((unsigned)(((int64_t)p.B * p.n * p.H + 7) / 8)), dim3(256), 0, st, p);
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
                        allow_smem<__nv_bfloat16, 192>(d), allow_smem<__nv_bfloat16, 256>(d)})
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
  return work_bytes(tree_splits(*dev, B, n, H, HK, D, n_ctx), B, n, H, D);
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
  if (a->n_ctx > 1 && a->kv_row == 0) return fail(BTF_ERR_ARG, "btf_tree_attention: the rows of k and v need a stride");
  if (!std::isfinite(a->scale)) return fail(BTF_ERR_ARG, "btf_tree_attention: scale must be finite");
  if (!a->work || reinterpret_cast<uintptr_t>(a->work) % 256 || a->work_bytes < 256)
    return fail(BTF_ERR_ARG, "btf_tree_attention: workspace null, not 256-byte aligned or too small");
  const DeviceInfo* dev = current_device();
  if (!dev) return BTF_ERR_STATE;
  const int splits = tree_splits(*dev, a->B, a->n, a->H, a->HK, a->D, a->n_ctx);
  if (a->work_bytes < work_bytes(splits, a->B, a->n, a->H, a->D))
    return fail(BTF_ERR_ARG, "btf_tree_attention: the workspace has %lld bytes, %lld are needed", (long long)a->work_bytes,
                (long long)work_bytes(splits, a->B, a->n, a->H, a->D));
  const bool b_one = a->B == 1 || a->kv_batch == 0, h_one = a->HK == 1 || a->kv_head == 0;
  CUtensorMap mk, mv;
  if (int rc = encode_kv(&mk, *a, a->k, b_one, h_one)) return rc;
  if (int rc = encode_kv(&mv, *a, a->v, b_one, h_one)) return rc;
  const TreeParams p{a->q, a->v, a->o, a->q_batch, a->q_node, a->q_head, a->kv_batch, a->kv_row, a->kv_head, a->o_batch,
                     a->o_node, a->o_head, a->B, a->n, a->H, a->HK, a->D, a->n_ctx,
                     (a->n * (a->H / a->HK) + kRowsM - 1) / kRowsM, splits, b_one ? 0 : 1, h_one ? 0 : 1, a->lens,
                     a->parents, a->counts, a->scale * 1.4426950408889634f, static_cast<float*>(a->work), dev->err_word};
  if ((int64_t)p.B * p.HK * p.splits * p.mtiles > INT32_MAX || (int64_t)p.B * p.n * p.H > ((int64_t)1 << 33))
    return fail(BTF_ERR_UNSUPPORTED, "btf_tree_attention: too many sequences and heads for one launch");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e =
      a->type == BTF_F16 ? launch_tree_d<__half>(mk, mv, p, st) : launch_tree_d<__nv_bfloat16>(mk, mv, p, st);
  return e == cudaSuccess ? BTF_OK : cuda_fail(e, "btf_tree_attention");
}

}  // extern "C"
