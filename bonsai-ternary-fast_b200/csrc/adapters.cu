// Low-rank adapters of many requests beside a shared projection (btf_adapters):
//
//   y_t = base_t + s_a B_a (A_a x_t),  a = the adapter of row t
//
// for up to three projections of the same rows (q, k and v; gate and up). Two
// launches: `shrink` makes h = A x (fp32), `expand` makes y. The rows are taken in
// tiles of one adapter, from a plan that sorts them (btf_adapter_plan).
//
// What bounds it: bytes. A row's x is read once, y written and base read once: with
// rank r that is 2 r (K + N) multiply-adds for (K + 2 N) elements, 64 a byte at r = 64
// in 16 bits, where the card has 250 a byte on tcgen05 and 80 on the warp-level MMA.
// For few rows the weights are what is read, once for the rows of an adapter, and there
// the time is the latency of one pass through memory after another. So the MMAs are
// warp-level (m16n8k16), whose operands come from global memory straight into
// registers, 16 bytes a lane: no shared memory, barrier or transposition lies between
// a load and its product, N, strides and row order are free, and the accumulators lie
// where y's rows are stored from.
//
// k is permuted alike in both operands of an MMA: the lane of place t holds the 8
// consecutive elements 8 t .. 8 t + 7 of a 32-wide step (one 16-byte load), which are
// its k pairs of two MMAs.
//
// fp32 stays fp32: an fp32 x meets bf16 weights as three bf16 terms (24 bits) and fp16
// weights as two tf32 terms (22 bits, weights exact); h, always fp32, is split into
// three bf16 terms for an fp32 y and two for a 16-bit one (16 bits: 2^-18 of an
// element, a 500th of y's own rounding), or two fp16 terms (22 bits) of h over a power
// of two of its row, which keeps fp16's range.
#include <algorithm>

#include "adapters_tc.cuh"

namespace btf {
namespace {

using namespace adapt;

constexpr int kThreads = 256, kExpand = 64;

// ------------------------------------------------------------------ plan
// One CTA. Warp w counts and later places its own stretch of the rows, so that the
// order within an adapter is that of the rows whatever runs first.
__global__ void __launch_bounds__(1024) adapter_plan_kernel(const int32_t* index, int T, int n, uint8_t* plan, PlanLayout at) {
  extern __shared__ int hist[];  // [32 warps][n + 1]
  __shared__ int total[BTF_ADAPTERS_MAX + 1], first[BTF_ADAPTERS_MAX + 1];
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, nb = n + 1;
  for (int i = tid; i < 32 * nb; i += 1024) hist[i] = 0;
  __syncthreads();
  const int per = ((T + 31) / 32 + 31) / 32 * 32, t0 = warp * per, t1 = min(T, t0 + per);
  int* mine = hist + warp * nb;
  auto each = [&](auto fn) {
    for (int b = t0; b < t1; b += 32) {
      const int t = b + lane;
      int a = t < t1 ? index[t] : -2;
      if (a != -2 && (a < 0 || a >= n)) a = n;
      const unsigned same = __match_any_sync(0xffffffffu, a);
      fn(t, a, same, __popc(same & ((1u << lane) - 1)));
      __syncwarp();
    }
  };
  each([&](int t, int a, unsigned same, int before) {
    if (t < t1 && before == 0) mine[a] += __popc(same);
  });
  __syncthreads();
  for (int a = tid; a < nb; a += 1024) {
    int sum = 0;
    for (int w = 0; w < 32; ++w) {
      const int c = hist[w * nb + a];
      hist[w * nb + a] = sum;
      sum += c;
    }
    total[a] = sum;
  }
  __syncthreads();
  int32_t* head = reinterpret_cast<int32_t*>(plan);
  if (warp < 3) {  // running sums over the adapters: rows, small tiles, large tiles
    const int size = warp == 0 ? 1 : warp == 1 ? kSmall : kLarge;
    Tile* tiles = reinterpret_cast<Tile*>(plan + (warp == 1 ? at.small : at.large));
    int sum = 0, rows = 0;
    for (int b = 0; b < nb; b += 32) {
      const int a = b + lane, c = a < nb ? total[a] : 0, k = (c + size - 1) / size;
      int s = k, r = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int q = __shfl_up_sync(0xffffffffu, s, o), v = __shfl_up_sync(0xffffffffu, r, o);
        if (lane >= o) s += q, r += v;
      }
      if (a < nb) {
        if (warp == 0) {
          first[a] = rows + r - c;
        } else {
          for (int i = 0; i < k; ++i)
            tiles[sum + s - k + i] = {a < n ? a : -1, rows + r - c + i * size, min(size, c - i * size), 0};
        }
      }
      sum += __shfl_sync(0xffffffffu, s, 31);
      rows += __shfl_sync(0xffffffffu, r, 31);
    }
    if (lane == 0) {
      if (warp == 0) head[0] = T, head[1] = n, head[4] = T - total[n];
      else head[1 + warp] = sum;
    }
  }
  __syncthreads();
  int32_t *order = reinterpret_cast<int32_t*>(plan + at.order), *owner = reinterpret_cast<int32_t*>(plan + at.owner);
  each([&](int t, int a, unsigned same, int before) {
    if (t < t1) order[first[a] + mine[a] + before] = t, owner[first[a] + mine[a] + before] = a;
    __syncwarp();
    if (t < t1 && before == 0) mine[a] += __popc(same);
  });
}

template <typename T>
__device__ __forceinline__ void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                      uint32_t b1) {
  if constexpr (std::is_same_v<T, __half>)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 ld16(const void* p, bool on) {
  return on ? __ldg(static_cast<const uint4*>(p)) : make_uint4(0, 0, 0, 0);
}
// 8 consecutive elements of x as the B operands of a step: TERMS x 4 words of 16-bit pairs, or (fp32 x, fp16 weights)
// 2 x 8 tf32 values.
template <typename TX, typename TW>
struct XFrag {
  static constexpr bool kF32 = std::is_same_v<TX, float>;
  static constexpr bool kTf32 = kF32 && std::is_same_v<TW, __half>;
  static constexpr int kTerms = !kF32 ? 1 : kTf32 ? 2 : 3;
  static constexpr int kLoads = kF32 ? 2 : 1;
};

// ------------------------------------------------------------------ shrink
// A CTA takes a tile's rows, one projection and one of `splits` stretches of K, which its warps share: RG groups of
// NT x 8 rows times 8 / RG stretches. The weights are the MMA's 16-row side (RT x 16 of them), the rows of x its 8-wide
// side. The stretches of K of one CTA meet in shared memory, in order; those of several in `expand`.
template <typename TX, typename TW, int RT, int NT, int RG>
__global__ void __launch_bounds__(kThreads, RT == 8 || (RT == 4 && XFrag<TX, TW>::kTf32) ? 1 : 2)
    adapter_shrink_kernel(const __grid_constant__ Params p) {
  using F = XFrag<TX, TW>;
  constexpr int KG = kThreads / 32 / RG, kRows = RG * NT * 8;
  extern __shared__ float red[];  // [KG][kRows][RT * 16 + 4]
  constexpr int kPitch = RT * 16 + 4;
  pdl_wait();
  pdl_launch_dependents();  // (behind the wait: `expand` reads the plan before its own)
  if (!plan_ok(p)) return;
  constexpr int kParts = RG == 1 ? 1 : kLarge / kRows;  // of a tile
  const int split = blockIdx.x % p.splits, seg = blockIdx.x / p.splits % p.nseg, part = blockIdx.x / (p.splits * p.nseg);
  const int ti = part / kParts;
  if (ti >= p.head[p.which]) return;
  Tile tile = p.tiles[ti];
  tile.begin += part % kParts * kRows;
  tile.count = min(tile.count - part % kParts * kRows, kRows);
  if (tile.adapter < 0 || tile.count <= 0) return;
  const int rank = rank_of(p, tile.adapter);
  if (rank == 0) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int rg = warp % RG, kg = warp / RG;
  const Seg& s = p.seg[seg];
  const int steps = (p.K + 31) / 32, ways = p.splits * KG;
  const int way = split * KG + kg, k0 = (int)((int64_t)way * steps / ways), k1 = (int)((int64_t)(way + 1) * steps / ways);
  const TW* a = static_cast<const TW*>(s.a) + tile.adapter * s.a_adapter + 8 * t;
  const TX* x[NT];
  bool on[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int r = (rg * NT + j) * 8 + g;
    on[j] = r < tile.count;
    x[j] = static_cast<const TX*>(p.x) + (on[j] ? p.order[tile.begin + r] * p.x_row : 0) + 8 * t;
  }
  float c[RT][NT][4];
#pragma unroll
  for (int m = 0; m < RT; ++m)
#pragma unroll
    for (int j = 0; j < NT; ++j) c[m][j][0] = c[m][j][1] = c[m][j][2] = c[m][j][3] = 0.f;
  const int mts = (rank + 15) / 16;
  if (rg * NT * 8 < tile.count) {
#pragma unroll 1
    for (int ks = k0; ks < k1; ++ks) {
      const int k = ks * 32;
      const bool kin = k + 8 * t < p.K;
      uint4 xw[NT][F::kLoads], lo[RT], hi[RT];
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int l = 0; l < F::kLoads; ++l) xw[j][l] = ld16(x[j] + k + 4 * l, kin && on[j]);
#pragma unroll
      for (int m = 0; m < RT; ++m) {
        lo[m] = ld16(a + (int64_t)(m * 16 + g) * s.a_row + k, kin && m < mts && m * 16 + g < p.R);
        hi[m] = ld16(a + (int64_t)(m * 16 + 8 + g) * s.a_row + k, kin && m < mts && m * 16 + 8 + g < p.R);
      }
      if constexpr (!F::kF32) {
#pragma unroll
        for (int m = 0; m < RT; ++m)
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            mma16<TW>(c[m][j], lo[m].x, hi[m].x, lo[m].y, hi[m].y, xw[j][0].x, xw[j][0].y);
            mma16<TW>(c[m][j], lo[m].z, hi[m].z, lo[m].w, hi[m].w, xw[j][0].z, xw[j][0].w);
          }
      } else if constexpr (!F::kTf32) {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const uint32_t w[8] = {xw[j][0].x, xw[j][0].y, xw[j][0].z, xw[j][0].w,
                                 xw[j][1].x, xw[j][1].y, xw[j][1].z, xw[j][1].w};
          uint32_t term[3][4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float v0 = __uint_as_float(w[2 * i]), v1 = __uint_as_float(w[2 * i + 1]);
            term[0][i] = __byte_perm(w[2 * i], w[2 * i + 1], 0x7632);  // cut off: never beyond fp32's range
            const float r0 = rest(v0, __uint_as_float(w[2 * i] & 0xffff0000u));
            const float r1 = rest(v1, __uint_as_float(w[2 * i + 1] & 0xffff0000u));
            term[1][i] = pack2<__nv_bfloat16>(r0, r1);
            const float2 mid = unpack2<__nv_bfloat16>(term[1][i]);
            term[2][i] = pack2<__nv_bfloat16>(r0 - mid.x, r1 - mid.y);
          }
#pragma unroll
          for (int e = 2; e >= 0; --e)
#pragma unroll
            for (int m = 0; m < RT; ++m) {
              mma16<TW>(c[m][j], lo[m].x, hi[m].x, lo[m].y, hi[m].y, term[e][0], term[e][1]);
              mma16<TW>(c[m][j], lo[m].z, hi[m].z, lo[m].w, hi[m].w, term[e][2], term[e][3]);
            }
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // the lane's elements 2 i and 2 i + 1
          uint32_t big[NT][2], small[NT][2];
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint4 v4 = xw[j][i >> 1];
              const uint32_t w = i & 1 ? (e ? v4.w : v4.z) : (e ? v4.y : v4.x);
              big[j][e] = w & 0xffffe000u;
              const float r = rest(__uint_as_float(w), __uint_as_float(big[j][e]));
              asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(small[j][e]) : "f"(r));
            }
#pragma unroll
          for (int m = 0; m < RT; ++m) {
            const uint32_t wl = i == 0 ? lo[m].x : i == 1 ? lo[m].y : i == 2 ? lo[m].z : lo[m].w;
            const uint32_t wh = i == 0 ? hi[m].x : i == 1 ? hi[m].y : i == 2 ? hi[m].z : hi[m].w;
            const float2 fl = unpack2<TW>(wl), fh = unpack2<TW>(wh);
            const uint32_t a0 = __float_as_uint(fl.x), a1 = __float_as_uint(fh.x), a2 = __float_as_uint(fl.y),
                           a3 = __float_as_uint(fh.y);
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              mma_tf32(c[m][j], a0, a1, a2, a3, small[j][0], small[j][1]);
              mma_tf32(c[m][j], a0, a1, a2, a3, big[j][0], big[j][1]);
            }
          }
        }
      }
    }
  }
  // c[m][j]: weight rows 16 m + g and + 8, rows 8 j + 2 t and + 1 of the group
  float* mine = red + (kg * kRows + rg * NT * 8) * kPitch;
#pragma unroll
  for (int m = 0; m < RT; ++m)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) mine[(j * 8 + 2 * t + (e & 1)) * kPitch + m * 16 + g + (e >> 1) * 8] = c[m][j][e];
  __syncthreads();
  const int quads = p.R / 4, live = min((rank + 3) / 4, quads);
  float* h = p.h + ((int64_t)(split * p.nseg + seg) * p.T + tile.begin) * p.R;
  for (int i = threadIdx.x; i < tile.count * quads; i += kThreads) {
    const int r = i / quads, q = i % quads;
    if (q >= live) continue;
    float4 v = *reinterpret_cast<const float4*>(red + r * kPitch + q * 4);
#pragma unroll
    for (int w = 1; w < KG; ++w) {
      const float4 u = *reinterpret_cast<const float4*>(red + (w * kRows + r) * kPitch + q * 4);
      v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
    }
    *reinterpret_cast<float4*>(h + (int64_t)r * p.R + q * 4) = v;
  }
}

// ------------------------------------------------------------------ expand
// Few rows: a CTA takes a tile's 16 rows and a stretch of the outputs of all projections, 32 at a time per warp. h's
// terms lie in shared memory as the MMA's A operands, 16 bytes a lane; the weights are its 8-wide side, with the rows of
// B so assigned that a lane ends up with 8 consecutive outputs of a row. (Prompts: adapters_tc.cu.)
template <typename TW, typename TY>
__global__ void __launch_bounds__(kExpand, 8) adapter_expand_kernel(const __grid_constant__ Params p) {
  constexpr bool kHalf = std::is_same_v<TW, __half>, kY32 = std::is_same_v<TY, float>;
  constexpr int kTerms = !kHalf && kY32 ? 3 : 2;
  constexpr int kRows = kSmall;
  constexpr int kYWords = 8 * (int)sizeof(TY) / 16;  // 16-byte words of a lane's 8 outputs
  extern __shared__ uint4 frag[];  // [k32 blocks][2][terms][32]
  __shared__ float mul[kRows];
  __shared__ int top[kRows];
  // The plan, the weights and base were complete before `shrink` let this grid start.
  // (A grid may only end after the one before it, or the one behind it starts too early: every way out waits.)
  pdl_launch_dependents();
  if (!plan_ok(p)) {
    pdl_wait();
    return;
  }
  const int range = blockIdx.x % p.ranges, ti = blockIdx.x / p.ranges;
  if (ti >= p.head[p.which]) {
    pdl_wait();
    return;
  }
  const Tile tile = p.tiles[ti];
  const int rank = tile.adapter < 0 ? 0 : rank_of(p, tile.adapter);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int blocks = (rank + 31) / 32;
  // the CTA's pieces, of all projections in a line
  auto pieces = [&](int i) { return (p.seg[i].N + kExpand - 1) / kExpand; };
  int total = 0;
  for (int i = 0; i < p.nseg; ++i) total += pieces(i);
  const int first = (int)((int64_t)range * total / p.ranges), last = (int)((int64_t)(range + 1) * total / p.ranges);
  int seg = 0, before = 0;  // pieces of the projections before seg
  int row[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) row[e] = e * 8 + g < tile.count ? p.order[tile.begin + e * 8 + g] : -1;
  bool waited = false;
  int have = -1;  // the projection whose h lies in shared memory
  for (int piece = first; piece < last; ++piece) {
    for (int k; piece - before >= (k = pieces(seg)); ++seg) before += k;
    const Seg& s = p.seg[seg];
    const int n0 = (piece - before) * kExpand + warp * 32;
    const bool copy = rank == 0;
    if (copy && s.base == s.y && s.base_row == s.y_row) continue;  // in place: stays
    // weights of the first k32 block and base on their way before h is looked at
    const TW* b = static_cast<const TW*>(s.b) + (copy ? 0 : tile.adapter * s.b_adapter) + 8 * t;
    auto load_b = [&](uint4 (&w)[4], int kb) {
      const int k = kb * 32 + 8 * t, valid = rank - k;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int n = n0 + 8 * (g >> 1) + 2 * j + (g & 1);
        w[j] = ld16(b + (int64_t)n * s.b_row + kb * 32, valid > 0 && n < s.N);
        if (valid > 0 && valid < 8) {  // columns behind the adapter's rank may hold anything
          uint32_t v[4] = {w[j].x, w[j].y, w[j].z, w[j].w};
#pragma unroll
          for (int i = 0; i < 4; ++i) v[i] &= valid >= 2 * i + 2 ? 0xffffffffu : valid == 2 * i + 1 ? 0xffffu : 0u;
          w[j] = make_uint4(v[0], v[1], v[2], v[3]);
        }
      }
    };
    uint4 wb[4];
    load_b(wb, 0);
    const int n8 = n0 + 8 * t;  // the lane's outputs
    uint4 bv[2][kYWords];
    const bool vec = s.vec && n8 + 8 <= s.N;
    if (s.base && vec) {
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int w = 0; w < kYWords; ++w)
          bv[e][w] = row[e] >= 0 ? *(reinterpret_cast<const uint4*>(static_cast<const TY*>(s.base) + row[e] * s.base_row + n8) + w)
                                 : make_uint4(0, 0, 0, 0);
    }
    if (!waited) {
      pdl_wait();
      waited = true;
    }
    if (have != seg && !copy) {
      __syncthreads();  // nobody reads the one before any more
      have = seg;
      const int chunks = blocks * 4;  // of 8 elements of h
      const float* h = p.h + ((int64_t)seg * p.T + tile.begin) * p.R;
      const int64_t next = (int64_t)p.nseg * p.T * p.R;
      auto sum = [&](int u, float (&v)[8]) {
        const int r = u / chunks, k = u % chunks * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.f;
        if (r >= tile.count || k >= rank) return;
        const float* from = h + (int64_t)r * p.R + k;
#pragma unroll 4
        for (int q = 0; q < p.splits; ++q, from += next) {
          const float4 v0 = ld_cg(from), v1 = ld_cg(from + 4);
          v[0] += v0.x, v[1] += v0.y, v[2] += v0.z, v[3] += v0.w;
          v[4] += v1.x, v[5] += v1.y, v[6] += v1.z, v[7] += v1.w;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (k + i >= rank) v[i] = 0.f;
      };
      if constexpr (kHalf) {  // each row over a power of two: its largest in [2^14, 2^15)
        for (int r = threadIdx.x; r < kRows; r += kExpand) top[r] = 0;
        __syncthreads();
        for (int u = threadIdx.x; u < kRows * chunks; u += kExpand) {
          float v[8];
          sum(u, v);
          float m = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(v[i]));
          atomicMax(&top[u / chunks], __float_as_int(m));
        }
        __syncthreads();
      }
      const float scale = p.scales ? p.scales[tile.adapter] : 1.f;
      for (int r = threadIdx.x; r < kRows; r += kExpand) {
        if constexpr (kHalf) {
          const int e = (top[r] >> 23) - 127;  // of the largest; 0, denormal and infinite rows stay as they are
          mul[r] = e >= -112 && e < 128 ? scale * __int_as_float((e - 14 + 127) << 23) : scale;
        } else {
          mul[r] = scale;
        }
      }
      for (int u = threadIdx.x; u < kRows * chunks; u += kExpand) {
        float v[8];
        sum(u, v);
        const int r = u / chunks, k = u % chunks;
        if constexpr (kHalf) {
          const int e = (top[r] >> 23) - 127;
          const float f = e >= -112 && e < 128 ? __int_as_float((14 - e + 127) << 23) : 1.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] *= f;
        }
        // row r of its 16: g = r % 8, words 0 and 2 (r < 8) or 1 and 3
        uint32_t* to = reinterpret_cast<uint32_t*>(frag + (k >> 2) * 2 * kTerms * 32 + (r & 7) * 4 + (k & 3)) + (r >> 3);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float v0 = v[2 * i], v1 = v[2 * i + 1];
#pragma unroll
          for (int e = 0; e < kTerms; ++e) {
            const uint32_t w = pack2<TW>(v0, v1);
            to[(((i >> 1) * kTerms + e) * 32) * 4 + (i & 1) * 2] = w;
            const float2 f = unpack2<TW>(w);
            v0 = rest(v0, f.x), v1 = rest(v1, f.y);
          }
        }
      }
      __syncthreads();
    }
    float c[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) c[j][0] = c[j][1] = c[j][2] = c[j][3] = 0.f;
#pragma unroll 1
    for (int kb = 0; kb < blocks; ++kb) {
      uint4 wn[4];
      if (kb + 1 < blocks) load_b(wn, kb + 1);
      const uint4* f = frag + (int64_t)kb * 2 * kTerms * 32 + lane;
#pragma unroll
      for (int e = kTerms - 1; e >= 0; --e) {
        const uint4 a0 = f[e * 32], a1 = f[(kTerms + e) * 32];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          mma16<TW>(c[j], a0.x, a0.y, a0.z, a0.w, wb[j].x, wb[j].y);
          mma16<TW>(c[j], a1.x, a1.y, a1.z, a1.w, wb[j].z, wb[j].w);
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) wb[j] = wn[j];
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      if (row[e] < 0) continue;
      const float f = copy ? 0.f : mul[e * 8 + g];
      float v[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[2 * j] = c[j][2 * e] * f, v[2 * j + 1] = c[j][2 * e + 1] * f;
      TY* y = static_cast<TY*>(s.y) + row[e] * s.y_row + n8;
      if (vec) {
        if (s.base) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if constexpr (kY32) {
              const uint4 w = bv[e][i >> 1];
              v[2 * i] += __uint_as_float(i & 1 ? w.z : w.x), v[2 * i + 1] += __uint_as_float(i & 1 ? w.w : w.y);
            } else {
              const uint4 w = bv[e][0];
              const float2 q = unpack2<TY>(i == 0 ? w.x : i == 1 ? w.y : i == 2 ? w.z : w.w);
              v[2 * i] += q.x, v[2 * i + 1] += q.y;
            }
          }
        }
        if constexpr (kY32) {
          reinterpret_cast<float4*>(y)[0] = make_float4(v[0], v[1], v[2], v[3]);
          reinterpret_cast<float4*>(y)[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
          *reinterpret_cast<uint4*>(y) = make_uint4(pack2<TY>(v[0], v[1]), pack2<TY>(v[2], v[3]), pack2<TY>(v[4], v[5]),
                                                    pack2<TY>(v[6], v[7]));
        }
      } else {
        const TY* base = s.base ? static_cast<const TY*>(s.base) + row[e] * s.base_row + n8 : nullptr;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (n8 + i < s.N) y[i] = from_f32<TY>(base ? v[i] + to_f32(base[i]) : v[i]);
      }
    }
  }
  if (!waited) pdl_wait();
}

// ------------------------------------------------------------------ launches
bool sizes_ok(int T, int K, int R, int nseg, int n) {
  return T >= 0 && T <= BTF_ADAPTERS_MAX_ROWS && K >= 8 && K % 8 == 0 && K <= (1 << 24) && R >= 8 && R % 8 == 0 &&
         R <= BTF_ADAPTERS_MAX_RANK && nseg >= 1 && nseg <= 3 && n >= 1 && n <= BTF_ADAPTERS_MAX;
}

// Tiles of 16 rows while the adapters' rows are few, of 128 for prompts.
struct Shape {
  bool large;
  int tiles;   // at most
  int splits;  // stretches of K
};
Shape shape_of(const DeviceInfo& d, int T, int K, int nseg, int n) {
  Shape s;
  s.large = T > 256;
  const int rows = s.large ? kLarge : kSmall;
  s.tiles = T / rows + std::min(n + 1, T);
  const int steps = (K + 31) / 32, warps = s.large ? 4 : 8;  // that share a CTA's stretch
  const int want = 2 * d.sm_count / (s.tiles * nseg * (s.large ? 2 : 1));
  s.splits = std::max(1, std::min({want, kMaxSplits, (steps + warps - 1) / warps}));
  return s;
}
// The workspace: h, and for prompts its terms and the rows' factors.
struct Work {
  int64_t terms, mul, bytes;
  Work(const Shape& s, int T, int R, int nseg) {
    terms = ((int64_t)s.splits * nseg * T * R * 4 + 15) / 16 * 16;
    mul = terms + (s.large ? (int64_t)3 * nseg * T * ((R + 63) / 64 * 64) * 2 : 0);
    bytes = mul + (s.large ? (int64_t)nseg * T * 4 : 0);
  }
};

template <typename TX, typename TW, int RT, int NT, int RG>
cudaError_t shrink(const Params& p, int tiles, cudaStream_t st, bool setup) {
  constexpr int smem = 8 / RG * (RG * NT * 8) * (RT * 16 + 4) * 4;
  if (setup)
    return cudaFuncSetAttribute(adapter_shrink_kernel<TX, TW, RT, NT, RG>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  return launch_pdl(adapter_shrink_kernel<TX, TW, RT, NT, RG>, dim3((unsigned)(tiles * p.nseg * p.splits * (RG == 1 ? 1 : kLarge / (RG * NT * 8)))), dim3(kThreads),
                    smem, st, p);
}
template <typename TX, typename TW, int RT>
cudaError_t shrink_rt(const Params& p, bool large, int tiles, cudaStream_t st, bool setup) {
  // 64 rows: 32 a warp where the accumulators leave room for it, else 16
  constexpr int NT = RT <= 4 && !std::is_same_v<TX, float> ? 4 : 2;
  if (setup)
    if (cudaError_t e = shrink<TX, TW, RT, 2, 1>(p, tiles, st, true)) return e;
  return large || setup ? shrink<TX, TW, RT, NT, 8 / NT>(p, tiles, st, setup) : shrink<TX, TW, RT, 2, 1>(p, tiles, st, false);
}
template <typename TX, typename TW>
cudaError_t shrink_r(const Params& p, bool large, int tiles, cudaStream_t st) {
  return p.R <= 16   ? shrink_rt<TX, TW, 1>(p, large, tiles, st, false)
         : p.R <= 32 ? shrink_rt<TX, TW, 2>(p, large, tiles, st, false)
         : p.R <= 64 ? shrink_rt<TX, TW, 4>(p, large, tiles, st, false)
                     : shrink_rt<TX, TW, 8>(p, large, tiles, st, false);
}
template <typename TX, typename TW>
cudaError_t shrink_setup() {
  const Params p{};
  for (cudaError_t e : {shrink_rt<TX, TW, 1>(p, true, 0, nullptr, true), shrink_rt<TX, TW, 2>(p, true, 0, nullptr, true),
                        shrink_rt<TX, TW, 4>(p, true, 0, nullptr, true), shrink_rt<TX, TW, 8>(p, true, 0, nullptr, true)})
    if (e != cudaSuccess) return e;
  return cudaSuccess;
}

template <typename TW, typename TY>
cudaError_t expand(Params p, int tiles, int sms, cudaStream_t st) {
  constexpr int terms = std::is_same_v<TW, __half> || !std::is_same_v<TY, float> ? 2 : 3;
  int64_t pieces = 0;
  for (int i = 0; i < p.nseg; ++i) pieces += (p.seg[i].N + kExpand - 1) / kExpand;
  p.ranges = (int)std::max<int64_t>(1, std::min<int64_t>(pieces, (8 * sms + tiles - 1) / tiles));
  return launch_pdl(adapter_expand_kernel<TW, TY>, dim3((unsigned)(tiles * p.ranges)), dim3(kExpand),
                    (size_t)(p.R + 31) / 32 * 2 * terms * 512, st, p);
}

}  // namespace

int adapters_setup(DeviceInfo& d) {
  const Params p{};
  if (32 * (BTF_ADAPTERS_MAX + 1) * 4 > d.optin_smem) return cuda_fail(cudaErrorInvalidValue, "adapter_plan_kernel attributes");
  for (cudaError_t e :
       {cudaFuncSetAttribute(adapter_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 32 * (BTF_ADAPTERS_MAX + 1) * 4),
        shrink_setup<float, __half>(), shrink_setup<float, __nv_bfloat16>(), shrink_setup<__half, __half>(),
        shrink_setup<__nv_bfloat16, __nv_bfloat16>()})
    if (e != cudaSuccess) return cuda_fail(e, "adapter kernels' attributes");
  return setup_tc();
}

}  // namespace btf

using namespace btf;

extern "C" {

int64_t btf_adapter_plan_bytes(int T, int n_adapters) {
  if (T < 0 || T > BTF_ADAPTERS_MAX_ROWS || n_adapters < 1 || n_adapters > BTF_ADAPTERS_MAX) {
    fail(BTF_ERR_ARG, "btf_adapter_plan_bytes: need T in 0..%d and 1..%d adapters (got %d, %d)", BTF_ADAPTERS_MAX_ROWS,
         BTF_ADAPTERS_MAX, T, n_adapters);
    return -1;
  }
  return PlanLayout(T, n_adapters).bytes;
}

int btf_adapter_plan(const int32_t* index, int T, int n_adapters, void* plan, int64_t plan_bytes, void* stream) {
  const int64_t bytes = btf_adapter_plan_bytes(T, n_adapters);
  if (bytes < 0) return BTF_ERR_ARG;
  if ((T > 0 && !index) || !plan || reinterpret_cast<uintptr_t>(plan) % 16)
    return fail(BTF_ERR_ARG, "btf_adapter_plan: null pointer, or a plan that is not 16-byte aligned");
  if (plan_bytes < bytes)
    return fail(BTF_ERR_ARG, "btf_adapter_plan: the plan has %lld bytes, %lld are needed", (long long)plan_bytes, (long long)bytes);
  if (!current_device()) return BTF_ERR_STATE;
  const cudaError_t e = launch_pdl(adapter_plan_kernel, dim3(1), dim3(1024), (size_t)32 * (n_adapters + 1) * 4,
                                   static_cast<cudaStream_t>(stream), index, T, n_adapters, static_cast<uint8_t*>(plan),
                                   PlanLayout(T, n_adapters));
  return e == cudaSuccess ? BTF_OK : cuda_fail(e, "btf_adapter_plan");
}

int64_t btf_adapters_work(int T, int K, int R, int nseg, int n_adapters) {
  if (!sizes_ok(T, K, R, nseg, n_adapters)) {
    fail(BTF_ERR_ARG, "btf_adapters_work: bad sizes (T %d, K %d, R %d, %d projections, %d adapters)", T, K, R, nseg, n_adapters);
    return -1;
  }
  const DeviceInfo* dev = current_device();
  if (!dev) return -1;
  return T == 0 ? 0 : Work(shape_of(*dev, T, K, nseg, n_adapters), T, R, nseg).bytes;
}

int btf_adapters(const btf_adapters_args* a, void* stream) {
  if (!a) return fail(BTF_ERR_ARG, "btf_adapters: null arguments");
  if (!sizes_ok(a->T, a->K, a->R, a->nseg, a->n_adapters))
    return fail(BTF_ERR_ARG,
                "btf_adapters: need T in 0..%d, K and R multiples of 8, R <= %d, 1..3 projections and 1..%d adapters (T %d, "
                "K %d, R %d, %d projections, %d adapters)",
                BTF_ADAPTERS_MAX_ROWS, BTF_ADAPTERS_MAX_RANK, BTF_ADAPTERS_MAX, a->T, a->K, a->R, a->nseg, a->n_adapters);
  if (a->w_type != BTF_F16 && a->w_type != BTF_BF16) return fail(BTF_ERR_ARG, "btf_adapters: the adapters are fp16 or bf16");
  if ((a->x_type != BTF_F32 && a->x_type != a->w_type) || (a->y_type != BTF_F32 && a->y_type != a->w_type))
    return fail(BTF_ERR_ARG, "btf_adapters: x and y are fp32 or of the adapters' type");
  if (a->T == 0) return BTF_OK;
  auto al = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  const int xb = elem_bytes(a->x_type), yb = elem_bytes(a->y_type);
  if (!a->x || !a->plan || !al(a->x) || !al(a->plan) || a->x_row < 0 || a->x_row * xb % 16)
    return fail(BTF_ERR_ARG, "btf_adapters: x or the plan is null or not 16-byte aligned, or x's rows are not");
  if (a->plan_bytes < PlanLayout(a->T, a->n_adapters).bytes)
    return fail(BTF_ERR_ARG, "btf_adapters: the plan is of other sizes (%lld bytes, %lld are needed)", (long long)a->plan_bytes,
                (long long)PlanLayout(a->T, a->n_adapters).bytes);
  Params p{};
  for (int i = 0; i < a->nseg; ++i) {
    const btf_adapter_seg& s = a->segs[i];
    if (s.N < 1 || s.N > 1 << 24) return fail(BTF_ERR_ARG, "btf_adapters: need 1 <= N <= 2^24 (got %d)", s.N);
    if (!s.a || !s.b || !s.y || !al(s.a) || !al(s.b))
      return fail(BTF_ERR_ARG, "btf_adapters: a, b or y is null, or a or b is not 16-byte aligned");
    for (int64_t v : {s.a_adapter, s.a_row, s.b_adapter, s.b_row})
      if (v < 0 || v % 8) return fail(BTF_ERR_ARG, "btf_adapters: the strides of a and b must be multiples of 8 elements, >= 0");
    if (s.a_row == 0 || (s.N > 1 && s.b_row == 0)) return fail(BTF_ERR_ARG, "btf_adapters: the rows of a and b need a stride");
    if (reinterpret_cast<uintptr_t>(s.y) % yb || reinterpret_cast<uintptr_t>(s.base) % yb)
      return fail(BTF_ERR_ARG, "btf_adapters: y or base is not aligned to its type");
    if (a->T > 1 && s.y_row < s.N) return fail(BTF_ERR_ARG, "btf_adapters: the rows of y overlap");
    if (s.base && s.base_row < 0) return fail(BTF_ERR_ARG, "btf_adapters: the stride of base is negative");
    if (s.base == s.y && a->T > 1 && s.base_row != s.y_row)
      return fail(BTF_ERR_ARG, "btf_adapters: in place needs the same strides");
    const int64_t y_row = a->T > 1 ? s.y_row : 0, base_row = a->T > 1 ? s.base_row : 0;
    const bool vec = al(s.y) && y_row * yb % 16 == 0 && al(s.base) && base_row * yb % 16 == 0;
    p.seg[i] = {s.a, s.b, s.base, s.y, s.a_adapter, s.a_row, s.b_adapter, s.b_row, base_row, y_row, s.N, vec};
  }
  const DeviceInfo* dev = current_device();
  if (!dev) return BTF_ERR_STATE;
  const Shape sh = shape_of(*dev, a->T, a->K, a->nseg, a->n_adapters);
  const Work w(sh, a->T, a->R, a->nseg);
  if (!a->work || !al(a->work) || a->work_bytes < w.bytes)
    return fail(BTF_ERR_ARG, "btf_adapters: workspace null, not 16-byte aligned or too small (%lld bytes, %lld are needed)",
                (long long)a->work_bytes, (long long)w.bytes);
  const PlanLayout at(a->T, a->n_adapters);
  const uint8_t* plan = static_cast<const uint8_t*>(a->plan);
  p.x = a->x, p.x_row = a->T > 1 ? a->x_row : 0;
  p.T = a->T, p.K = a->K, p.R = a->R, p.n = a->n_adapters, p.nseg = a->nseg, p.splits = sh.splits, p.ranges = 1;
  p.ranks = a->ranks, p.scales = a->scales;
  p.head = reinterpret_cast<const int32_t*>(plan), p.order = reinterpret_cast<const int32_t*>(plan + at.order);
  p.owner = reinterpret_cast<const int32_t*>(plan + at.owner);
  p.tiles = reinterpret_cast<const Tile*>(plan + (sh.large ? at.large : at.small)), p.which = sh.large ? 3 : 2;
  uint8_t* work = static_cast<uint8_t*>(a->work);
  p.h = reinterpret_cast<float*>(work), p.terms = reinterpret_cast<uint16_t*>(work + w.terms), p.mul = reinterpret_cast<float*>(work + w.mul);
  p.err = dev->err_word;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool half = a->w_type == BTF_F16, x32 = a->x_type == BTF_F32, y32 = a->y_type == BTF_F32;
  cudaError_t e = half ? (x32 ? shrink_r<float, __half>(p, sh.large, sh.tiles, st) : shrink_r<__half, __half>(p, sh.large, sh.tiles, st))
                       : (x32 ? shrink_r<float, __nv_bfloat16>(p, sh.large, sh.tiles, st)
                              : shrink_r<__nv_bfloat16, __nv_bfloat16>(p, sh.large, sh.tiles, st));
  if (e == cudaSuccess && sh.large) return expand_tc(p, half, y32, dev->sm_count, st);
  if (e == cudaSuccess)
    e = half ? (y32 ? expand<__half, float>(p, sh.tiles, dev->sm_count, st) : expand<__half, __half>(p, sh.tiles, dev->sm_count, st))
             : (y32 ? expand<__nv_bfloat16, float>(p, sh.tiles, dev->sm_count, st)
                    : expand<__nv_bfloat16, __nv_bfloat16>(p, sh.tiles, dev->sm_count, st));
  return e == cudaSuccess ? BTF_OK : cuda_fail(e, "btf_adapters");
}

}  // extern "C"
