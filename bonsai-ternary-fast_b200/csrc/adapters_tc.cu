// Low-rank adapters of prompts (btf_adapters with many rows), on the tcgen05 tensor
// cores: y = base + s B h for tiles of 128 rows of one adapter.
//
// What bounds it: y's and base's bytes. An element of y takes 2 r operations for each
// term of h (see adapters.cu), 256 at r = 64 in bf16: 0.15 ps of a card that moves the
// element's 4 bytes, base and y, in 0.61. So the MMAs (128 x 128 outputs at a time, four accumulators in tensor memory)
// run far ahead and the kernel is its way out: 8 warps, each with 32 rows of every other
// tile. A lane has a row: copies bring 256 bytes of its base into shared memory ahead of
// their turn and take the sum from the same place to y: one TMA copy of 32 rows x 128
// bytes where the rows follow one another (a prompt's do), else 16 bytes a lane, eight
// lanes a row. (Bulk copies of a row each are issued one after another by a warp: 178 us
// for what takes 105 so: 6007 rows of 17408 in bf16 on a base, 418 MB, 4 TB/s.)
//
// Rows that begin anywhere (an odd width, rows of y that are not 16-byte aligned), which neither kind of copy takes, go
// through registers, 32 outputs of a row by the lanes of a warp: 3655 rows of 2533 and 10797 among them 222 us, 610 with
// base read row by row; these instructions, not bytes, are the time there.
//
// Work: the tiles of 128 rows times 128 outputs of all projections make a line, cut into
// equal stretches of one CTA per SM. Warp 8 brings the terms of the rows' h (made by a
// small kernel between) and the weights by TMA, warp 9 issues the MMAs.
#include <cuda.h>

#include "adapters_tc.cuh"
#include "tcgen05.cuh"

namespace btf {
namespace adapt {
namespace {

using namespace tc;

constexpr int kCols = 128, kEpi = 8, kThreads = (kEpi + 2) * 32, kBufs = 4;
constexpr uint64_t kWaitNs = 1000000000ull;
constexpr int kBlock = 128 * 128;          // bytes of 128 rows x 64 elements
constexpr int kUnit = 128;                 // bytes of a row that move at once
constexpr int kSlot = 32 * kUnit;           // a warp's rows, 128-byte swizzle

struct ExpandMaps {
  CUtensorMap h, b[3], y[3], base[3];
};
struct ExpandParams : Params {
  int b_mul[3];  // 0: every adapter has the same B
  int wide[3];   // rows of y (and base) take bulk copies
  int blocks;                    // 64-wide blocks of R
  int stages, hs, slots;         // slots of the weights, of h, of a warp
};
struct Misc {
  uint64_t full[2], empty[2], acc_full[kBufs], acc_empty[kBufs], h_full[2], h_empty[2], final, base[kEpi][3];
  uint32_t tmem;
  int abort;
};
static_assert(kLarge == 128 && sizeof(Misc) <= 512);

// The present tile of the line.
struct Line {
  int pieces[3], total;  // 128-wide pieces of each projection and of a row tile
  __device__ __forceinline__ explicit Line(const Params& p) {
    total = 0;
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      pieces[i] = i < p.nseg ? (p.seg[i].N + kCols - 1) / kCols : 0;
      total += pieces[i];
    }
  }
  // Row tile, projection and piece of `at`; the piece's last neighbour of the same projection is at `end`.
  __device__ __forceinline__ void place(int at, int& ti, int& seg, int& piece, int& end) const {
    ti = at / total;
    piece = at - ti * total;
    seg = 0;
    if (piece >= pieces[0]) piece -= pieces[0], seg = 1;
    if (seg == 1 && piece >= pieces[1]) piece -= pieces[1], seg = 2;
    end = at + (seg == 0 ? pieces[0] : seg == 1 ? pieces[1] : pieces[2]) - piece;
  }
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, int x, int y, uint32_t src) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(reinterpret_cast<uint64_t>(map)),
               "r"(x), "r"(y), "r"(src)
               : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

__device__ __forceinline__ float ld_cg1(const float* p) {  // behind the wait, as ld_cg
  float v;
  asm volatile("ld.global.cg.f32 %0, [%1];" : "=f"(v) : "l"(p) : "memory");
  return v;
}

// ------------------------------------------------------------------ terms
// h summed over the stretches of K, cut to the adapter's rank and split into terms [TERMS][nseg][T][wide], and the
// factor of each row: its adapter's scale, over the power of two that fp16 terms carry. Eight lanes a row.
template <typename TW, int TERMS>
__global__ void __launch_bounds__(256) adapter_terms_kernel(const __grid_constant__ Params p, uint16_t* terms, int wide) {
  pdl_wait();
  pdl_launch_dependents();  // (behind the wait: the next grid reads the plan before its own)
  const int at = blockIdx.x * 32 + (threadIdx.x >> 3), l = threadIdx.x & 7, seg = blockIdx.y;
  if (p.head[0] != p.T || p.head[1] != p.n) return;
  const bool live = at < p.head[4];  // rows with an adapter come first
  const int a = live ? p.owner[at] : 0, rank = live ? rank_of(p, a) : 0, splits = long_splits(p);
  const int64_t next = (int64_t)p.nseg * p.T * p.R;
  const float* h = p.h + ((int64_t)seg * p.T + at) * p.R;
  float v[2][8];  // of a row's 128 at most: elements 8 l .. and 64 + 8 l ..
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    const int k = b * 64 + l * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[b][i] = 0.f;
    if (k >= rank) continue;
    const float* from = h + k;
#pragma unroll 4
    for (int q = 0; q < splits; ++q, from += next) {
      const float4 v0 = ld_cg(from), v1 = ld_cg(from + 4);
      v[b][0] += v0.x, v[b][1] += v0.y, v[b][2] += v0.z, v[b][3] += v0.w;
      v[b][4] += v1.x, v[b][5] += v1.y, v[b][6] += v1.z, v[b][7] += v1.w;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (k + i >= rank) v[b][i] = 0.f;
  }
  const float scale = live && p.scales ? p.scales[a] : 1.f;
  float f = 1.f, back = scale;
  if constexpr (std::is_same_v<TW, __half>) {  // the row over a power of two: its largest in [2^14, 2^15)
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = fmaxf(m, fmaxf(fabsf(v[0][i]), fabsf(v[1][i])));
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const int e = (__float_as_int(m) >> 23) - 127;  // 0, denormal and infinite rows stay as they are
    if (e >= -112 && e < 128) f = __int_as_float((14 - e + 127) << 23), back = scale * __int_as_float((e - 14 + 127) << 23);
  }
  if (!live) return;
  if (l == 0) p.mul[(int64_t)seg * p.T + at] = back;
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    if (b * 64 >= wide) break;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[b][i] *= f;
#pragma unroll
    for (int e = 0; e < TERMS; ++e) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float v0 = v[b][2 * i], v1 = v[b][2 * i + 1];
        w[i] = !std::is_same_v<TW, __half> && e == 0 ? pack2<TW>(in_bf16(v0), in_bf16(v1)) : pack2<TW>(v0, v1);
        const float2 u = unpack2<TW>(w[i]);
        v[b][2 * i] = rest(v0, u.x), v[b][2 * i + 1] = rest(v1, u.y);
      }
      *reinterpret_cast<uint4*>(terms + (((int64_t)e * p.nseg + seg) * p.T + at) * wide + b * 64 + l * 8) =
          make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

// ------------------------------------------------------------------ y
template <typename TW, typename TY>
__global__ void __launch_bounds__(kThreads, 1)
    adapter_expand_tc_kernel(const __grid_constant__ ExpandMaps maps, const __grid_constant__ ExpandParams p) {
  constexpr bool kHalf = std::is_same_v<TW, __half>, kY32 = std::is_same_v<TY, float>, kBf16 = !kHalf;
  constexpr int kTerms = !kHalf && kY32 ? 3 : 2;
  constexpr int kWidth = kUnit / (int)sizeof(TY), kUnits = kCols / kWidth;  // outputs of a unit, units of a tile's row
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw), sbase = (raw + 1023) & ~1023u;
  uint8_t* smem = smem_raw + (sbase - raw);
  const uint32_t h_bytes = kTerms * p.blocks * kBlock, off_ring = p.hs * h_bytes, off_slots = off_ring + p.stages * p.blocks * kBlock;
  const uint32_t off_misc = off_slots + kEpi * p.slots * kSlot;
  Misc& ms = *reinterpret_cast<Misc*>(smem + off_misc);
  volatile int* abort_flag = &ms.abort;
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  if (warp == kEpi + 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ms.tmem)),
                 "r"((uint32_t)(kBufs * kCols))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&ms.full[i]), 1), mbar_init(smem_u32(&ms.empty[i]), 1);
      mbar_init(smem_u32(&ms.h_full[i]), 1), mbar_init(smem_u32(&ms.h_empty[i]), 1);
    }
    for (int i = 0; i < kBufs; ++i) mbar_init(smem_u32(&ms.acc_full[i]), 1), mbar_init(smem_u32(&ms.acc_empty[i]), 4);
    mbar_init(smem_u32(&ms.final), 1);
    for (int i = 0; i < kEpi; ++i)
      for (int k = 0; k < 3; ++k) mbar_init(smem_u32(&ms.base[i][k]), 1);
    ms.abort = 0;
    fence_mbar_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, ms.tmem, 0);
  // The plan, the weights and base were complete before `terms` let this grid start; h is what the wait is for.
  pdl_launch_dependents();

  auto wait = [&](const uint64_t& bar, uint32_t parity) -> bool {  // bounded
    const uint32_t a = smem_u32(&bar);
    if (mbar_try_wait(a, parity)) return true;
    if (*abort_flag) return false;
    if (mbar_wait_bounded(a, parity, kWaitNs)) return true;
    atomicCAS(p.err, 0, kErrWaitTimeout);
    *abort_flag = 1;
    return false;
  };
  auto warp_wait = [&](const uint64_t& bar, uint32_t parity) -> bool { return __all_sync(0xffffffffu, wait(bar, parity)); };

  const Line line(p);
  int first = 0, last = 0;
  if (plan_ok(p)) {
    const int64_t all = (int64_t)p.head[p.which] * line.total;
    first = (int)(all * blockIdx.x / gridDim.x), last = (int)(all * (blockIdx.x + 1) / gridDim.x);
  }
  // Every role walks the same runs (row tile, projection) and counts the tiles with an adapter: t.
  int t = 0, run = 0;
  bool ok = true;
  if (warp == kEpi) {
    // ---------------------------------------------------------- weights
    if (lane == 0) {
      int sent = 0;
      bool waited = false;
      for (int at = first; ok && at < last;) {
        int ti, seg, piece, end;
        line.place(at, ti, seg, piece, end);
        end = min(end, last);
        const Tile tile = p.tiles[ti];
        const int rank = tile.adapter < 0 ? 0 : rank_of(p, tile.adapter), blocks = (rank + 63) / 64;
        if (rank == 0) {
          at = end;
          continue;
        }
        for (int begin = at; ok && at < end; ++at, ++piece, ++t) {
          const int s = t % p.stages;
          if (t >= p.stages && !(ok = wait(ms.empty[s], (uint32_t)((t / p.stages - 1) & 1)))) break;
          const uint32_t bar = smem_u32(&ms.full[s]), dst = sbase + off_ring + s * p.blocks * kBlock;
          mbar_expect_tx(bar, blocks * kBlock);
          for (int k = 0; k < blocks; ++k)
            tma_load_3d(dst + k * kBlock, &maps.b[seg], k * 64, piece * kCols, tile.adapter * p.b_mul[seg], bar);
          ++sent;
          if (at > begin) continue;
          // with the run's first weights: its rows' h
          if (!waited) {
            pdl_wait();
            asm volatile("fence.proxy.async.global;" ::: "memory");  // h was written as ordinary stores
          }
          waited = true;
          const int hs = run % p.hs;
          if (run >= p.hs && !(ok = wait(ms.h_empty[hs], (uint32_t)((run / p.hs - 1) & 1)))) break;
          const uint32_t hbar = smem_u32(&ms.h_full[hs]);
          mbar_expect_tx(hbar, kTerms * blocks * kBlock);
          for (int e = 0; e < kTerms; ++e)
            for (int k = 0; k < blocks; ++k)
              tma_load_3d(sbase + hs * h_bytes + (e * p.blocks + k) * kBlock, &maps.h, k * 64, tile.begin, e * p.nseg + seg, hbar);
          ++run;
        }
      }
      // after a time-out, leave no copy in flight into this CTA's shared memory (bounded)
      if (!ok || *abort_flag) {
        for (int k = max(0, sent - p.stages); k < sent; ++k)
          mbar_wait_bounded(smem_u32(&ms.full[k % p.stages]), (uint32_t)((k / p.stages) & 1), kWaitNs / 10);
        for (int k = max(0, run - p.hs); k < run; ++k)
          mbar_wait_bounded(smem_u32(&ms.h_full[k % p.hs]), (uint32_t)((k / p.hs) & 1), kWaitNs / 10);
      }
    }
  } else if (warp == kEpi + 1) {
    // ---------------------------------------------------------- MMAs
    constexpr uint32_t kDesc = idesc_f16(kBf16, false, 128, kCols);
    for (int at = first; ok && at < last;) {
      int ti, seg, piece, end;
      line.place(at, ti, seg, piece, end);
      end = min(end, last);
      const Tile tile = p.tiles[ti];
      const int rank = tile.adapter < 0 ? 0 : rank_of(p, tile.adapter), steps = (rank + 15) / 16;
      if (rank == 0) {
        at = end;
        continue;
      }
      const int hs = run % p.hs;
      ok = warp_wait(ms.h_full[hs], (uint32_t)((run++ / p.hs) & 1));
      for (; ok && at < end; ++at, ++t) {
        const int s = t % p.stages, buf = t % kBufs;
        if (!(ok = warp_wait(ms.full[s], (uint32_t)((t / p.stages) & 1)))) break;
        if (t >= kBufs && !(ok = warp_wait(ms.acc_empty[buf], (uint32_t)((t / kBufs - 1) & 1)))) break;
        const uint32_t ws = sbase + off_ring + s * p.blocks * kBlock;
        if (rank & 15) {
          // columns behind the rank may hold anything, and 0 x NaN is NaN: those of the last step are cleared
          for (int r = lane; r < kCols; r += 32) {
            uint8_t* row = smem + (ws - sbase) + (rank >> 6) * kBlock + r * 128;
            for (int c = rank & 63; c < ((rank & 63) + 15) / 16 * 16; ++c)
              *reinterpret_cast<uint16_t*>(row + (((c >> 3) ^ (r & 7)) << 4) + (c & 7) * 2) = 0;
          }
          fence_proxy_async_smem();
          __syncwarp();
        }
        tc_fence_after();
        if (elect_one()) {
          const uint32_t d = tmem + buf * kCols;
          // (all steps of the lower terms before those of the first: the sum is cut off at its own size each time)
#pragma unroll
          for (int e = kTerms - 1; e >= 0; --e)
#pragma unroll 1
            for (int k = 0; k < steps; ++k) {
              const uint32_t off = (k >> 2) * kBlock + (k & 3) * 32;
              mma_f16_ss(d, smem_desc_sw128(sbase + hs * h_bytes + e * p.blocks * kBlock + off), smem_desc_sw128(ws + off), kDesc,
                         k > 0 || e < kTerms - 1);
            }
          if (at + 1 == end) mma_commit(smem_u32(&ms.h_empty[hs]));
          mma_commit(smem_u32(&ms.empty[s]));
          mma_commit(smem_u32(&ms.acc_full[buf]));
        }
        __syncwarp();
      }
    }
    if (elect_one()) mma_commit(smem_u32(&ms.final));  // completes when every MMA issued above has finished
    __syncwarp();
    mbar_wait_bounded(smem_u32(&ms.final), 0, kWaitNs);
    __syncwarp();
  } else {
    // ---------------------------------------------------------- the way out: 32 rows a warp, every other tile
    // A group takes every other one of the tiles with an adapter, by their number t, so that an accumulator is always the same
    // group's, which waits for each of its phases in turn: a wait tells a phase only from the one before it.
    const int group = warp >> 2, r = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t own_at = off_slots + warp * p.slots * kSlot;  // the warp's slots
    bool waited = false;
    int q = 0;        // units so far, of which each has its slot in turn
    uint32_t loads = 0, pending = 0;  // bit i: the phase of slot i's next load; whether one is under way
    for (int at = first; at < last;) {
      int ti, seg, piece, end;
      line.place(at, ti, seg, piece, end);
      end = min(end, last);
      const Tile tile = p.tiles[ti];
      const int rank = tile.adapter < 0 ? 0 : rank_of(p, tile.adapter);
      const Seg& s = p.seg[seg];
      const bool copy = rank == 0, live = r < tile.count, wide = p.wide[seg];
      const int rows = min(32, tile.count - (warp & 3) * 32);  // of the warp
      if (copy && s.base == s.y && s.base_row == s.y_row) {  // in place: stays
        at = end;
        continue;
      }
      const int64_t row = live ? p.order[tile.begin + r] : 0;
      const bool base = s.base != nullptr;
      const int row0 = (int)__shfl_sync(0xffffffffu, row, 0);
      const bool tiled = wide && rows >= 32 && __all_sync(0xffffffffu, row == row0 + lane);
      int rows_at[8];  // of the lane's words where the rows do not follow one another
#pragma unroll
      for (int i = 0; i < 8; ++i) rows_at[i] = (int)__shfl_sync(0xffffffffu, row, i * 4 + (lane >> 3));
      // bytes of a row of the unit from output n0 that copies move; 0: rows that begin anywhere, and odd ends
      auto bytes_of = [&](int n0) {
        // (a TMA copy stops at N, but a store only between 16-byte words: it would write zeros to the end of N's)
        const int b = min(kUnit, (s.N - n0) * (int)sizeof(TY));
        return !wide || b <= 0 || b % 16 ? 0 : tiled ? kUnit : b;
      };
      const int start = at + (((copy ? at : t) ^ group) & 1), units = start < end ? ((end - start + 1) >> 1) * kUnits : 0;
      const int first_n = (piece + start - at) * kCols;  // the run's first output of this group
      auto output = [&](int u) { return first_n + u / kUnits * 2 * kCols + u % kUnits * kWidth; };
      // base of the run's unit u to its slot, which its last store has been read from
      auto fetch = [&](int u, int qu) {
        const int n0 = output(u), b = u < units && base && rows > 0 ? bytes_of(n0) : 0, slot = qu % p.slots;
        const uint32_t to = sbase + own_at + slot * kSlot;
        if (b && tiled) {
          const uint32_t bar = smem_u32(&ms.base[warp][slot]);
          pending |= 1u << slot;
          if (lane == 0) {
            mbar_expect_tx(bar, kSlot);
            tma_load_2d(to, &maps.base[seg], n0, row0, bar);
          }
        } else if (b && (lane & 7) * 16 < b) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int k = i * 4 + (lane >> 3);
            if (k < rows)
              cp_async16(to + k * kUnit + (((lane & 7) ^ (k & 7)) << 4),
                         static_cast<const TY*>(s.base) + rows_at[i] * s.base_row + n0 + (lane & 7) * (16 / (int)sizeof(TY)));
          }
        }
        cp_commit();  // (a group a unit, empty or not)
      };
      bulk_wait_read();
      fence_proxy_async_smem();  // (what lay in the slots by ordinary stores; in a run those come behind its last bulk copy)
      __syncwarp();
      for (int u = 0; u < p.slots - 1; ++u) fetch(u, q + u);
      if (!waited) {
        pdl_wait();
        waited = true;
      }
      const float mul = copy || !live ? 0.f : ld_cg1(p.mul + (int64_t)seg * p.T + tile.begin + r);
      int u = 0;
      for (; at < end; ++at) {
        const int now = t;
        t += !copy;
        if (((copy ? at : now) & 1) != group) continue;
        const int buf = now % kBufs;
        if (!copy) {
          ok = ok && warp_wait(ms.acc_full[buf], (uint32_t)((now / kBufs) & 1));
          tc_fence_after();
        }
#pragma unroll 1  // (its code has to stay in its cache)
        for (int h = 0; h < kUnits; ++h, ++u, ++q) {
          const int n0 = output(u), bytes = bytes_of(n0), slot = q % p.slots;
          uint8_t* own = smem + own_at + slot * kSlot;
          // into the slot of the unit before, whose store has been read
          bulk_wait_read();
          __syncwarp();
          fetch(u + p.slots - 1, q + p.slots - 1);
          if (base && bytes && rows > 0) {
            if (tiled) {
              ok = ok && warp_wait(ms.base[warp][slot], (loads >> slot) & 1);
              if (ok) loads ^= 1u << slot, pending &= ~(1u << slot);
            } else {
              if (p.slots == 3) cp_wait<2>();
              else cp_wait<1>();
              __syncwarp();
            }
          }
#pragma unroll
          for (int c = 0; c < kWidth / 32; ++c) {
            uint32_t v[32];
            if (!copy) {
              tmem_ld32(tmem + buf * kCols + h * kWidth + c * 32 + lanes, v);
              tmem_wait_ld(v);
            } else {
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = 0;
            }
            if (c == kWidth / 32 - 1 && h == kUnits - 1 && !copy) {
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(smem_u32(&ms.acc_empty[buf]));
            }
            if (!ok || rows <= 0) continue;
            if (bytes) {
#pragma unroll
              for (int w = 0; w < 2 * (int)sizeof(TY); ++w) {
                const int k = c * 2 * (int)sizeof(TY) + w;  // the row's 16-byte word
                uint4* mine = reinterpret_cast<uint4*>(own + lane * kUnit + ((k ^ (lane & 7)) << 4));
                const uint4 b4 = base ? *mine : make_uint4(0, 0, 0, 0);
                const uint32_t b[4] = {b4.x, b4.y, b4.z, b4.w};
                uint32_t o[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  if constexpr (kY32) {
                    o[i] = __float_as_uint(fmaf(__uint_as_float(v[w * 4 + i]), mul, __uint_as_float(b[i])));
                  } else {
                    const float2 b2 = unpack2<TY>(b[i]);
                    o[i] = pack2<TY>(fmaf(__uint_as_float(v[w * 8 + 2 * i]), mul, b2.x),
                                     fmaf(__uint_as_float(v[w * 8 + 2 * i + 1]), mul, b2.y));
                  }
                }
                *mine = make_uint4(o[0], o[1], o[2], o[3]);
              }
            } else if (n0 + c * 32 < s.N) {
              // rows that begin anywhere, and odd ends: a row at a time for the warp
              float* stage = reinterpret_cast<float*>(own);
#pragma unroll
              for (int i = 0; i < 32; ++i) stage[lane * 32 + (i ^ lane)] = __uint_as_float(v[i]) * mul;
              __syncwarp();
              TY* const to = static_cast<TY*>(s.y);
              const TY* const from = static_cast<const TY*>(s.base);
              const int n = n0 + c * 32 + lane;
              TY had[32];  // (all of base on its way before the first store, which it might lie behind otherwise)
#pragma unroll
              for (int k = 0; k < 32; ++k) {
                const int64_t at_row = __shfl_sync(0xffffffffu, row, k);
                if (from && k < rows && n < s.N) had[k] = from[at_row * s.base_row + n];
              }
#pragma unroll
              for (int k = 0; k < 32; ++k) {
                const int64_t at_row = __shfl_sync(0xffffffffu, row, k);
                if (k < rows && n < s.N) {
                  const float o = stage[k * 32 + (lane ^ k)];
                  to[at_row * s.y_row + n] = from_f32<TY>(from ? o + to_f32(had[k]) : o);
                }
              }
              __syncwarp();
            }
          }
          if (bytes && ok) {
            fence_proxy_async_smem();
            __syncwarp();
            if (tiled) {
              if (lane == 0) tma_store_2d(&maps.y[seg], n0, row0, sbase + own_at + slot * kSlot);
            } else if ((lane & 7) * 16 < bytes) {
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const int k = i * 4 + (lane >> 3);
                if (k < rows)
                  *reinterpret_cast<uint4*>(static_cast<TY*>(s.y) + rows_at[i] * s.y_row + n0 + (lane & 7) * (16 / (int)sizeof(TY))) =
                      *reinterpret_cast<const uint4*>(own + k * kUnit + (((lane & 7) ^ (k & 7)) << 4));
              }
            }
            bulk_commit();
          }
        }
      }
    }
    bulk_wait();
    cp_wait<0>();
    // after a time-out, leave no copy in flight into this CTA's shared memory (bounded)
    for (int i = 0; i < p.slots; ++i)
      if ((pending >> i) & 1) mbar_wait_bounded(smem_u32(&ms.base[warp][i]), (loads >> i) & 1, kWaitNs / 10);
    if (!waited) pdl_wait();  // (a grid may only end after the one before it)
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kEpi + 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)(kBufs * kCols)) : "memory");
  }
}

// What fits: the terms of h twice, two slots of weights and three of each warp, or less where there are three terms or
// R > 64.
int expand_smem(int R, int terms, ExpandParams* p) {
  p->blocks = (R + 63) / 64;
  p->hs = p->blocks == 1 ? 2 : 1;
  p->stages = p->blocks == 1 || terms == 2 ? 2 : 1;
  p->slots = p->blocks == 1 && terms == 2 ? 3 : 2;
  return 1024 + (p->hs * terms + p->stages) * p->blocks * kBlock + kEpi * p->slots * kSlot + 512;
}

// b as [adapters][N][R]
int encode_b(CUtensorMap* m, const Params& p, int seg, bool half, bool one) {
  const Seg& s = p.seg[seg];
  const cuuint64_t dims[3] = {(cuuint64_t)p.R, (cuuint64_t)s.N, (cuuint64_t)(one ? 1 : p.n)};
  const cuuint64_t strides[2] = {(cuuint64_t)(s.N > 1 ? s.b_row * 2 : 16), (cuuint64_t)(one ? 16 : s.b_adapter * 2)};
  const cuuint32_t box[3] = {64, kCols, 1}, step[3] = {1, 1, 1};
  const CUresult r = encode_fn()(m, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(s.b),
                        dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? BTF_OK : fail(BTF_ERR_ARG, "btf_adapters: the strides of b make no tensor map (%d)", (int)r);
}

// y or base as [T][N], 32 rows x 128 bytes at a time
int encode_y(CUtensorMap* m, const Params& p, const void* at, int64_t row, int N, bool y32, bool half) {
  const cuuint64_t dims[2] = {(cuuint64_t)N, (cuuint64_t)p.T}, strides[1] = {(cuuint64_t)(row * (y32 ? 4 : 2))};
  const cuuint32_t box[2] = {y32 ? 32u : 64u, 32}, step[2] = {1, 1};
  const CUresult r = encode_fn()(m, y32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                                 2, const_cast<void*>(at), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                 CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? BTF_OK : fail(BTF_ERR_ARG, "btf_adapters: the strides of y or base make no tensor map (%d)", (int)r);
}

template <typename TW, typename TY>
cudaError_t expand(const ExpandMaps& maps, ExpandParams p, int sms, cudaStream_t st, bool setup) {
  constexpr int terms = std::is_same_v<TW, __half> || !std::is_same_v<TY, float> ? 2 : 3;
  if (setup)
    return cudaFuncSetAttribute(adapter_expand_tc_kernel<TW, TY>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                std::max(expand_smem(BTF_ADAPTERS_MAX_RANK, terms, &p), expand_smem(64, terms, &p)));
  const int smem = expand_smem(p.R, terms, &p);
  if (cudaError_t e = launch_pdl(adapter_terms_kernel<TW, terms>, dim3((unsigned)((p.T + 31) / 32), p.nseg), dim3(256), 0, st, p, p.terms,
                                 p.blocks * 64))
    return e;
  return launch_pdl(adapter_expand_tc_kernel<TW, TY>, dim3((unsigned)sms), dim3(kThreads), (size_t)smem, st, maps, p);
}

}  // namespace

int setup_tc() {
  const ExpandMaps m{};
  const ExpandParams p{};
  for (cudaError_t e : {expand<__half, float>(m, p, 0, nullptr, true), expand<__half, __half>(m, p, 0, nullptr, true),
                        expand<__nv_bfloat16, float>(m, p, 0, nullptr, true),
                        expand<__nv_bfloat16, __nv_bfloat16>(m, p, 0, nullptr, true)})
    if (e != cudaSuccess) return cuda_fail(e, "adapter kernels' attributes");
  return BTF_OK;
}

// h's terms as [terms x nseg][T][wide]
int encode_h(CUtensorMap* m, const Params& p, int terms, bool half) {
  const int wide = (p.R + 63) / 64 * 64;
  const cuuint64_t dims[3] = {(cuuint64_t)wide, (cuuint64_t)p.T, (cuuint64_t)(terms * p.nseg)};
  const cuuint64_t strides[2] = {(cuuint64_t)wide * 2, (cuuint64_t)wide * 2 * p.T};
  const cuuint32_t box[3] = {64, kLarge, 1}, step[3] = {1, 1, 1};
  const CUresult r = encode_fn()(m, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, p.terms, dims,
                                 strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                 CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? BTF_OK : fail(BTF_ERR_CUDA, "btf_adapters: no tensor map of the workspace (%d)", (int)r);
}

int expand_tc(const Params& q, bool half, bool y32, int sms, cudaStream_t st) {
  if (!encode_fn()) return fail(BTF_ERR_CUDA, "btf_adapters: cuTensorMapEncodeTiled is not available");
  ExpandMaps maps{};
  ExpandParams p{};
  static_cast<Params&>(p) = q;
  for (int i = 0; i < p.nseg; ++i) {
    const Seg& s = p.seg[i];
    const bool one = p.n == 1 || s.b_adapter == 0;
    p.b_mul[i] = !one;
    if (int rc = encode_b(&maps.b[i], p, i, half, one)) return rc;
    // one row of base for all rows (stride 0) makes no map, nor do rows that begin anywhere
    p.wide[i] = s.vec && (!s.base || s.base_row > 0);
    if (p.wide[i]) {
      if (int rc = encode_y(&maps.y[i], p, s.y, s.y_row, s.N, y32, half)) return rc;
      if (s.base)
        if (int rc = encode_y(&maps.base[i], p, s.base, s.base_row, s.N, y32, half)) return rc;
    }
  }
  if (int rc = encode_h(&maps.h, p, half || !y32 ? 2 : 3, half)) return rc;
  const cudaError_t e = half ? (y32 ? expand<__half, float>(maps, p, sms, st, false) : expand<__half, __half>(maps, p, sms, st, false))
                             : (y32 ? expand<__nv_bfloat16, float>(maps, p, sms, st, false)
                                    : expand<__nv_bfloat16, __nv_bfloat16>(maps, p, sms, st, false));
  return e == cudaSuccess ? BTF_OK : cuda_fail(e, "btf_adapters");
}

}  // namespace adapt
}  // namespace btf
