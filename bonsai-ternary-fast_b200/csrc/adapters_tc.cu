// Low-rank adapters of prompts (btf_adapters with many rows), on the tcgen05 tensor
// cores: y = base + s B h for tiles of 128 rows of one adapter.
//
// What bounds it: y's and base's bytes. An element of y takes 2 r multiply-adds for each
// term of h (see adapters.cu), 256 at r = 64 in bf16: 0.06 ns of a card that moves 4 bytes
// in 0.6. So the MMAs (128 x 128 outputs at a time, four accumulators in tensor memory)
// run far ahead and the kernel is its way out: 8 warps, each with 32 rows of every other
// tile, read base two tiles before they need it, whole 32-byte sectors of a row a lane,
// add and store as many at a time.
//
// Work: the tiles of 128 rows times 128 outputs of all projections make a line, cut into
// equal stretches of one CTA per SM. A stretch begins with the terms of its rows' h in
// shared memory (the A operand, 128-byte swizzle) and again where it comes to other rows
// or another projection. Warp 8 brings the weights by TMA, warp 9 issues the MMAs.
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
constexpr int kStagePitch = 33;            // a warp's 32 x 32 outputs on their way, in words
constexpr int kStageBytes = kEpi * 32 * kStagePitch * 4;

struct ExpandMaps {
  CUtensorMap b[3];
};
struct ExpandParams : Params {
  int b_mul[3];  // 0: every adapter has the same B
  int wide[3];   // y (and base) take whole 32-byte words
  int blocks, stages;  // 64-wide blocks of R; slots of the ring
};
struct Misc {
  uint64_t full[4], empty[4], acc_full[kBufs], acc_empty[kBufs], h_ready, final;
  uint32_t tmem;
  int abort;
  float mul[2][kLarge];  // of this run's rows, and the next one's
};
static_assert(kLarge == 128 && sizeof(Misc) <= 2048);

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

__device__ __forceinline__ void ld_v8(uint32_t (&v)[8], const void* p) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
               : "l"(p));
}
__device__ __forceinline__ void st_v8(void* p, const uint32_t (&v)[8]) {
  asm volatile("st.global.v8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
               "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "l"(p)
               : "memory");
}

template <typename TW, typename TY>
__global__ void __launch_bounds__(kThreads, 1)
    adapter_expand_tc_kernel(const __grid_constant__ ExpandMaps maps, const __grid_constant__ ExpandParams p) {
  constexpr bool kHalf = std::is_same_v<TW, __half>, kY32 = std::is_same_v<TY, float>, kBf16 = !kHalf;
  constexpr int kTerms = !kHalf && kY32 ? 3 : 2;
  constexpr int kWords = 32 / (int)sizeof(TY);      // outputs of a 32-byte word
  constexpr int kPer = 32 / kWords;                 // of which 32 outputs have so many
  constexpr int kRing = kY32 ? 2 : 4;               // base: so many 32-wide pieces ahead
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw), sbase = (raw + 1023) & ~1023u;
  uint8_t* smem = smem_raw + (sbase - raw);
  const uint32_t off_ring = kTerms * p.blocks * kBlock, off_misc = off_ring + p.stages * p.blocks * kBlock;
  Misc& ms = *reinterpret_cast<Misc*>(smem + off_misc);
  float* stage = reinterpret_cast<float*>(smem + off_misc + 2048);
  volatile int* abort_flag = &ms.abort;
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  if (warp == kEpi + 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ms.tmem)),
                 "r"((uint32_t)(kBufs * kCols))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (tid == 0) {
    for (int i = 0; i < 4; ++i) mbar_init(smem_u32(&ms.full[i]), 1), mbar_init(smem_u32(&ms.empty[i]), 1);
    for (int i = 0; i < kBufs; ++i) mbar_init(smem_u32(&ms.acc_full[i]), 1), mbar_init(smem_u32(&ms.acc_empty[i]), 4);
    mbar_init(smem_u32(&ms.h_ready), kEpi);
    mbar_init(smem_u32(&ms.final), 1);
    ms.abort = 0;
    fence_mbar_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, ms.tmem, 0);
  // The plan, the weights and base were complete before `shrink` let this grid start.
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
        for (; ok && at < end; ++at, ++piece, ++t) {
          const int s = t % p.stages;
          if (t >= p.stages && !(ok = wait(ms.empty[s], (uint32_t)((t / p.stages - 1) & 1)))) break;
          const uint32_t bar = smem_u32(&ms.full[s]), dst = sbase + off_ring + s * p.blocks * kBlock;
          mbar_expect_tx(bar, blocks * kBlock);
          for (int k = 0; k < blocks; ++k)
            tma_load_3d(dst + k * kBlock, &maps.b[seg], k * 64, piece * kCols, tile.adapter * p.b_mul[seg], bar);
          ++sent;
        }
      }
      // after a time-out, leave no copy in flight into this CTA's shared memory (bounded)
      if (!ok || *abort_flag)
        for (int k = max(0, sent - p.stages); k < sent; ++k)
          mbar_wait_bounded(smem_u32(&ms.full[k % p.stages]), (uint32_t)((k / p.stages) & 1), kWaitNs / 10);
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
      ok = warp_wait(ms.h_ready, (uint32_t)(run++ & 1));
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
#pragma unroll 1
          for (int k = 0; k < steps; ++k) {
            const uint32_t off = (k >> 2) * kBlock + (k & 3) * 32;
            const uint64_t bd = smem_desc_sw128(ws + off);
#pragma unroll
            for (int e = kTerms - 1; e >= 0; --e)
              mma_f16_ss(d, smem_desc_sw128(sbase + e * p.blocks * kBlock + off), bd, kDesc, k > 0 || e < kTerms - 1);
          }
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
    const int group = warp >> 2, r = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    float* own = stage + warp * 32 * kStagePitch;
    bool waited = false;
    for (int at = first; at < last;) {
      int ti, seg, piece, end;
      line.place(at, ti, seg, piece, end);
      end = min(end, last);
      const Tile tile = p.tiles[ti];
      const int rank = tile.adapter < 0 ? 0 : rank_of(p, tile.adapter);
      const Seg& s = p.seg[seg];
      const bool copy = rank == 0, live = r < tile.count, wide = p.wide[seg];
      if (copy && s.base == s.y && s.base_row == s.y_row) {  // in place: stays
        at = end;
        continue;
      }
      const int64_t row = live ? p.order[tile.begin + r] : 0;
      TY* y = static_cast<TY*>(s.y) + row * s.y_row;
      const TY* base = s.base ? static_cast<const TY*>(s.base) + row * s.base_row : nullptr;
      auto whole = [&](int pc) { return wide && (pc + 1) * kCols <= s.N; };  // a piece that takes 32-byte words
      // base of the 32-wide pieces ahead of the group's
      uint32_t ring[kRing][kPer][8];
      auto fetch = [&](uint32_t (&v)[kPer][8], int pc, int c) {
        if (base && live && whole(pc)) {
#pragma unroll
          for (int w = 0; w < kPer; ++w) ld_v8(v[w], base + pc * kCols + c * 32 + w * kWords);
        }
      };
      const int mine = at + ((at ^ group) & 1);  // the group's first
#pragma unroll
      for (int c = 0; c < kRing; ++c)
        if (mine < end) fetch(ring[c], piece + mine - at, c);
      if (!waited) {
        pdl_wait();
        waited = true;
      }
      float mul = 0.f;
      if (!copy) {
        // this run's h, in terms, where the MMAs of the one before are done: two threads a row
        if (t > 0) ok = ok && warp_wait(ms.acc_full[(t - 1) % kBufs], (uint32_t)(((t - 1) / kBufs) & 1));
        const int hr = tid >> 1, chunks = (rank + 15) / 16 * 2;  // of 8 elements
        const float* h = p.h + ((int64_t)seg * p.T + tile.begin + hr) * p.R;
        const int64_t next = (int64_t)p.nseg * p.T * p.R;
        auto sum = [&](int k, float (&v)[8]) {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = 0.f;
          if (hr >= tile.count || k * 8 >= rank) return;
          const float* from = h + k * 8;
#pragma unroll 4
          for (int q = 0; q < p.splits; ++q, from += next) {
            const float4 v0 = ld_cg(from), v1 = ld_cg(from + 4);
            v[0] += v0.x, v[1] += v0.y, v[2] += v0.z, v[3] += v0.w;
            v[4] += v1.x, v[5] += v1.y, v[6] += v1.z, v[7] += v1.w;
          }
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (k * 8 + i >= rank) v[i] = 0.f;
        };
        const float scale = p.scales ? p.scales[tile.adapter] : 1.f;
        float f = 1.f, back = scale;
        if constexpr (kHalf) {  // the row over a power of two: its largest in [2^14, 2^15)
          float m = 0.f;
          for (int k = tid & 1; k < chunks; k += 2) {
            float v[8];
            sum(k, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(v[i]));
          }
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
          const int e = (__float_as_int(m) >> 23) - 127;  // 0, denormal and infinite rows stay as they are
          if (e >= -112 && e < 128) f = __int_as_float((14 - e + 127) << 23), back = scale * __int_as_float((e - 14 + 127) << 23);
        }
        if ((tid & 1) == 0) ms.mul[run & 1][hr] = back;
        for (int k = tid & 1; k < chunks; k += 2) {
          float v[8];
          sum(k, v);
          uint8_t* to = smem + (k >> 3) * kBlock + hr * 128 + (((k & 7) ^ (hr & 7)) << 4);
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] *= f;
#pragma unroll
          for (int e = 0; e < kTerms; ++e) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              w[i] = pack2<TW>(v[2 * i], v[2 * i + 1]);
              const float2 u = unpack2<TW>(w[i]);
              v[2 * i] = rest(v[2 * i], u.x), v[2 * i + 1] = rest(v[2 * i + 1], u.y);
            }
            *reinterpret_cast<uint4*>(to + e * p.blocks * kBlock) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&ms.h_ready));
        asm volatile("bar.sync 1, 256;" ::: "memory");  // mul; every run, by every warp of these
        mul = ms.mul[run++ & 1][r];
      }
      for (; at < end; ++at, ++piece) {
        const int now = t;
        t += !copy;
        if ((at & 1) != group) continue;
        const int buf = now % kBufs;
        if (!copy) {
          ok = ok && warp_wait(ms.acc_full[buf], (uint32_t)((now / kBufs) & 1));
          tc_fence_after();
        }
        const bool fast = whole(piece);
#pragma unroll
        for (int c = 0; c < kCols / 32; ++c) {
          uint32_t v[32];
          if (!copy) {
            tmem_ld32(tmem + buf * kCols + c * 32 + lanes, v);
            tmem_wait_ld(v);
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = 0;
          }
          if (c == kCols / 32 - 1 && !copy) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&ms.acc_empty[buf]));
          }
          if (!ok) continue;
          if (fast) {
            uint32_t (&q)[kPer][8] = ring[c % kRing];
            if (live) {
#pragma unroll
              for (int w = 0; w < kPer; ++w) {
                uint32_t o[8];
                if constexpr (kY32) {
#pragma unroll
                  for (int i = 0; i < 8; ++i)
                    o[i] = __float_as_uint(fmaf(__uint_as_float(v[w * 8 + i]), mul, base ? __uint_as_float(q[w][i]) : 0.f));
                } else {
#pragma unroll
                  for (int i = 0; i < 8; ++i) {
                    const float2 b2 = base ? unpack2<TY>(q[w][i]) : make_float2(0.f, 0.f);
                    o[i] = pack2<TY>(fmaf(__uint_as_float(v[w * 16 + 2 * i]), mul, b2.x),
                                     fmaf(__uint_as_float(v[w * 16 + 2 * i + 1]), mul, b2.y));
                  }
                }
                st_v8(y + piece * kCols + c * 32 + w * kWords, o);
              }
            }
          } else {
            // rows that begin anywhere, and the last outputs: through shared memory, a row at a time for the warp
#pragma unroll
            for (int i = 0; i < 32; ++i) own[lane * kStagePitch + i] = __uint_as_float(v[i]) * mul;
            __syncwarp();
            const int n = piece * kCols + c * 32 + lane;
#pragma unroll 4
            for (int k = 0; k < 32; ++k) {
              const int64_t kr = __shfl_sync(0xffffffffu, row, k);
              if ((warp & 3) * 32 + k < tile.count && n < s.N) {
                const float o = own[k * kStagePitch + lane];
                static_cast<TY*>(s.y)[kr * s.y_row + n] =
                    from_f32<TY>(s.base ? o + to_f32(static_cast<const TY*>(s.base)[kr * s.base_row + n]) : o);
              }
            }
            __syncwarp();
          }
          // the next 32-wide piece that this place of the ring is for
          const int ahead = c + kRing < kCols / 32 ? 0 : 2;
          if (at + ahead < end) fetch(ring[c % kRing], piece + ahead, (c + kRing) % (kCols / 32));
        }
      }
    }
    if (!waited) pdl_wait();  // (a grid may only end after the one before it)
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kEpi + 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)(kBufs * kCols)) : "memory");
  }
}

int expand_smem(int R, int terms, int* blocks, int* stages) {
  *blocks = (R + 63) / 64;
  *stages = *blocks == 1 ? 4 : 2;
  return 1024 + (terms + *stages) * *blocks * kBlock + 2048 + kStageBytes;
}

// b as [adapters][N][R]
int encode_b(CUtensorMap* m, const Params& p, int seg, bool half, bool one) {
  const EncodeFn fn = encode_fn();
  if (!fn) return fail(BTF_ERR_CUDA, "btf_adapters: cuTensorMapEncodeTiled is not available");
  const Seg& s = p.seg[seg];
  const cuuint64_t dims[3] = {(cuuint64_t)p.R, (cuuint64_t)s.N, (cuuint64_t)(one ? 1 : p.n)};
  const cuuint64_t strides[2] = {(cuuint64_t)(s.N > 1 ? s.b_row * 2 : 16), (cuuint64_t)(one ? 16 : s.b_adapter * 2)};
  const cuuint32_t box[3] = {64, kCols, 1}, step[3] = {1, 1, 1};
  const CUresult r = fn(m, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(s.b),
                        dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? BTF_OK : fail(BTF_ERR_ARG, "btf_adapters: the strides of b make no tensor map (%d)", (int)r);
}

template <typename TW, typename TY>
cudaError_t expand(const ExpandMaps& maps, ExpandParams p, int sms, cudaStream_t st, bool setup) {
  constexpr int terms = std::is_same_v<TW, __half> || !std::is_same_v<TY, float> ? 2 : 3;
  const int smem = expand_smem(setup ? BTF_ADAPTERS_MAX_RANK : p.R, terms, &p.blocks, &p.stages);
  if (setup)
    return cudaFuncSetAttribute(adapter_expand_tc_kernel<TW, TY>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                std::max(smem, expand_smem(64, terms, &p.blocks, &p.stages)));
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

int expand_tc(const Params& q, bool half, bool y32, int sms, cudaStream_t st) {
  ExpandMaps maps{};
  ExpandParams p{};
  static_cast<Params&>(p) = q;
  const int size = y32 ? 4 : 2;
  for (int i = 0; i < p.nseg; ++i) {
    const Seg& s = p.seg[i];
    const bool one = p.n == 1 || s.b_adapter == 0;
    p.b_mul[i] = !one;
    p.wide[i] = reinterpret_cast<uintptr_t>(s.y) % 32 == 0 && s.y_row * size % 32 == 0 &&
                reinterpret_cast<uintptr_t>(s.base) % 32 == 0 && s.base_row * size % 32 == 0;
    if (int rc = encode_b(&maps.b[i], p, i, half, one)) return rc;
  }
  const cudaError_t e = half ? (y32 ? expand<__half, float>(maps, p, sms, st, false) : expand<__half, __half>(maps, p, sms, st, false))
                             : (y32 ? expand<__nv_bfloat16, float>(maps, p, sms, st, false)
                                    : expand<__nv_bfloat16, __nv_bfloat16>(maps, p, sms, st, false));
  return e == cudaSuccess ? BTF_OK : cuda_fail(e, "btf_adapters");
}

}  // namespace adapt
}  // namespace btf
