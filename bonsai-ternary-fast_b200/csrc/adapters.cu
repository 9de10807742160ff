// Low-rank adapters of many requests beside a shared projection (btf_adapters):
//
//   y_t = base_t + s_a B_a (A_a x_t),  a = the adapter of row t
//
// for up to three projections of the same rows (q, k and v; gate and up). The rows are
// taken in tiles of one adapter, from a plan that sorts them (btf_adapter_plan). Few
// rows: tiles of 16 and two launches, `shrink` makes h = A x (fp32), `expand` makes y.
// Prompts: tiles of 128 rows, `shrink`, a small kernel that lays h out as operands, and y
// on tcgen05 (adapters_tc.cu).
//
// What bounds it: bytes. A row's x is read once, y written and base read once: with
// rank r that is 2 r (K + N) operations for (K + 2 N) elements, 32 to 64 a byte at r = 64
// in 16 bits, where the card has 250 a byte on tcgen05 and 80 on the warp-level MMA.
// (An fp32 x takes three times the MMAs, and its terms have to be made: prompts of it are
// bound by the issue of these, 60 % of the slots and 37 % of the tensor pipe: 6007 rows of
// 8 requests, 5120 to q, k and v, rank 64: 242 us, of which the bytes take 79.)
// For few rows the weights are what is read, once for the rows of an adapter, and there
// the time is the latency of one pass through memory after another: 1 fp32 row, 6144 to
// 5120, rank 16: 8.1 us (0.3 MB); 200 fp16 rows over 9 adapters, 1672 to 4091, rank 24:
// 12 us; 48 fp32 rows over 24 adapters, 5120 to q, k and v, rank 64: 18.9 us (39 MB,
// 2.1 TB/s). `expand` can start under `shrink`, but at rank 64 two CTAs of that take the
// registers of an SM, so most of it comes behind. The MMAs there are warp-level
// (m16n8k16), whose operands come from global memory straight into registers, 16 bytes a lane: no shared memory, barrier or
// transposition lies between a load and its product, N, strides and row order are free,
// and the accumulators lie where y's rows are stored from. `expand` reads what does not
// depend on h before it waits for it, and a piece's weights and base under the piece
// before.
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
//
// The tensor cores cut a sum off, by up to 2^-23 of its size towards 0 in every MMA, where
// fp32 additions round. So the products of an fp32 x are summed there over 32 of K only,
// the lower terms first, and those sums by fp32 additions: 6007 rows of 17408, rank 64, against
// 64 bits: 2.2e-7 of y's root mean square (1.0e-5 with one tensor-core sum over a stretch of K,
// for up to 4 % less time; rows of 5120: 1.7e-7 and 3.0e-6). A 16-bit x keeps to one: 1.6e-6
// there in an fp32 y, where sums over 32 would cost 2 to 25 % of the call.
#include <algorithm>

#include "adapters_tc.cuh"

namespace btf {
namespace {

using namespace adapt;

constexpr int kThreads = 256, kExpand = 64;

// ------------------------------------------------------------------ plan
// One CTA. Warp w counts and later places its own stretch of the rows, so that the
// order within an adapter is that of the rows whatever runs first.
//
// What bounds it: chains of reads, and the tiles of an adapter, T / 16 and T / 128 of them, that one lane
// lists: 48 rows of 24 adapters 2.8 us, 6007 rows 7.2 (all of one adapter 17.7), 100000 rows 91 (263); of 1024
// adapters, whose counters 32 warps have each, 15 to 19 for up to 1024 rows, 22 for 6007. Once a step.
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
    Tile* large = reinterpret_cast<Tile*>(plan + at.large);
    SmallTile* small = reinterpret_cast<SmallTile*>(plan + at.small);
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
          for (int i = 0; i < k; ++i) {
            const Tile tile{a < n ? a : -1, rows + r - c + i * size, min(size, c - i * size), 0};
            if (warp == 1) small[sum + s - k + i].tile = tile;
            else large[sum + s - k + i] = tile;
          }
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
  // where each adapter's small tiles begin
  if (warp == 0) {
    int sum = 0;
    for (int b = 0; b < nb; b += 32) {
      const int a = b + lane, k = a < nb ? (total[a] + kSmall - 1) / kSmall : 0;
      int s = k;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int q = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += q;
      }
      if (a < nb) total[a] = sum + s - k;
      sum += __shfl_sync(0xffffffffu, s, 31);
    }
  }
  __syncthreads();
  SmallTile* small = reinterpret_cast<SmallTile*>(plan + at.small);
  int32_t *order = reinterpret_cast<int32_t*>(plan + at.order), *owner = reinterpret_cast<int32_t*>(plan + at.owner);
  each([&](int t, int a, unsigned same, int before) {
    if (t < t1) {
      const int i = mine[a] + before;  // the row's place among its adapter's
      order[first[a] + i] = t, owner[first[a] + i] = a;
      small[total[a] + i / kSmall].rows[i % kSmall] = t;
    }
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
__device__ __forceinline__ uint4 ld16(const void* p, bool on) {  // of weights
  return on ? __ldg(static_cast<const uint4*>(p)) : make_uint4(0, 0, 0, 0);
}
// of x, which the kernel before may still have been writing when this one started: not a read-only load
__device__ __forceinline__ uint4 ld16_x(const void* p, bool on) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (on) asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
// 8 consecutive elements of NT rows of x as the B operands of a 32-wide step: `kTerms` terms of 4 words of 16-bit pairs,
// or (fp32 x, fp16 weights) 2 terms of 8 tf32 values.
template <typename TX, typename TW, int NT>
struct XTerms {
  static constexpr bool kF32 = std::is_same_v<TX, float>;
  static constexpr bool kTf32 = kF32 && std::is_same_v<TW, __half>;
  static constexpr int kTerms = !kF32 ? 1 : kTf32 ? 2 : 3, kWords = kTf32 ? 8 : 4;
  static constexpr int kLoads = kF32 ? 2 : 1;
  uint32_t v[NT][kTerms][kWords];

  __device__ __forceinline__ explicit XTerms(const uint4 (&xw)[NT][kLoads]) {
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      uint32_t w[4 * kLoads];
#pragma unroll
      for (int l = 0; l < kLoads; ++l) w[4 * l] = xw[j][l].x, w[4 * l + 1] = xw[j][l].y, w[4 * l + 2] = xw[j][l].z, w[4 * l + 3] = xw[j][l].w;
      if constexpr (!kF32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[j][0][i] = w[i];
      } else if constexpr (!kTf32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float v0 = __uint_as_float(w[2 * i]), v1 = __uint_as_float(w[2 * i + 1]);
          v[j][0][i] = __byte_perm(w[2 * i], w[2 * i + 1], 0x7632);  // cut off: never beyond fp32's range
          const float r0 = rest(v0, __uint_as_float(w[2 * i] & 0xffff0000u));
          const float r1 = rest(v1, __uint_as_float(w[2 * i + 1] & 0xffff0000u));
          v[j][1][i] = pack2<__nv_bfloat16>(r0, r1);
          const float2 mid = unpack2<__nv_bfloat16>(v[j][1][i]);
          v[j][2][i] = pack2<__nv_bfloat16>(r0 - mid.x, r1 - mid.y);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          v[j][0][i] = w[i] & 0xffffe000u;
          // (at fp32's last exponent cut to 11 bits, not rounded up to 2^128 with the first)
          float r = rest(__uint_as_float(w[i]), __uint_as_float(v[j][0][i]));
          asm("min.NaN.xorsign.abs.f32 %0, %0, %1;" : "+f"(r) : "f"(0x1.ffcp116f));
          asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(v[j][1][i]) : "f"(r));
        }
      }
    }
  }
  // `products` of an fp32 x into sums of their own, which c takes by fp32 additions (see the top).
  template <int RT>
  __device__ __forceinline__ void add(float (&c)[RT][NT][4], const uint4 (&lo)[RT], const uint4 (&hi)[RT], int ms, int ns) const {
    if constexpr (!kF32) {
      products(c, lo, hi, ms, ns);
    } else {
      constexpr int MB = RT < 2 ? RT : 2;  // (registers)
#pragma unroll
      for (int m0 = 0; m0 < RT; m0 += MB) {
        float d[MB][NT][4];
        uint4 l[MB], h[MB];
#pragma unroll
        for (int m = 0; m < MB; ++m) {
          l[m] = lo[m0 + m], h[m] = hi[m0 + m];
#pragma unroll
          for (int j = 0; j < NT; ++j) d[m][j][0] = d[m][j][1] = d[m][j][2] = d[m][j][3] = 0.f;
        }
        products(d, l, h, ms - m0, ns);
#pragma unroll
        for (int m = 0; m < MB; ++m)
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) c[m0 + m][j][e] += d[m][j][e];
      }
    }
  }
  // c += the products: lo and hi the weights' rows g and g + 8 of each 16; of the weights' 16s and the rows' 8s only the
  // first ms and ns have anything.
  template <int RT>
  __device__ __forceinline__ void products(float (&c)[RT][NT][4], const uint4 (&lo)[RT], const uint4 (&hi)[RT], int ms, int ns) const {
    if constexpr (!kTf32) {
#pragma unroll
      for (int e = kTerms - 1; e >= 0; --e) {
#pragma unroll
        for (int m = 0; m < RT; ++m)
#pragma unroll
          for (int j = 0; j < NT; ++j)
            if (m < ms && j < ns) mma16<TW>(c[m][j], lo[m].x, hi[m].x, lo[m].y, hi[m].y, v[j][e][0], v[j][e][1]);
#pragma unroll
        for (int m = 0; m < RT; ++m)
#pragma unroll
          for (int j = 0; j < NT; ++j)
            if (m < ms && j < ns) mma16<TW>(c[m][j], lo[m].z, hi[m].z, lo[m].w, hi[m].w, v[j][e][2], v[j][e][3]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)  // the lane's elements 2 i and 2 i + 1
#pragma unroll
        for (int m = 0; m < RT; ++m) {
          if (m >= ms) break;
          const float2 fl = unpack2<TW>(i == 0 ? lo[m].x : i == 1 ? lo[m].y : i == 2 ? lo[m].z : lo[m].w);
          const float2 fh = unpack2<TW>(i == 0 ? hi[m].x : i == 1 ? hi[m].y : i == 2 ? hi[m].z : hi[m].w);
#pragma unroll
          for (int e = 1; e >= 0; --e)
#pragma unroll
            for (int j = 0; j < NT; ++j)
              if (j < ns)
                mma_tf32(c[m][j], __float_as_uint(fl.x), __float_as_uint(fh.x), __float_as_uint(fl.y), __float_as_uint(fh.y),
                         v[j][e][2 * i], v[j][e][2 * i + 1]);
        }
    }
  }
};

// ------------------------------------------------------------------ shrink
// Few rows: a CTA takes a tile's 16 rows, one projection and one of `splits` stretches of K, which its warps share. The
// weights are the MMA's 16-row side (RT x 16 of them), the rows of x its 8-wide side. The stretches of K of one CTA meet in
// shared memory, in order; those of several in `expand`.
template <typename TX, typename TW, int RT>
__global__ void __launch_bounds__(kThreads, RT == 8 || (RT == 4 && XTerms<TX, TW, 2>::kTf32) ? 1 : 2)
    adapter_shrink_kernel(const __grid_constant__ Params p) {
  // (fp32: the terms of 8 rows at a time, whose making overlaps the MMAs of the 8 before)
  constexpr int NT = 2, JT = std::is_same_v<TX, float> ? 1 : 2;
  using F = XTerms<TX, TW, JT>;
  constexpr int KG = kThreads / 32, kRows = kSmall;
  extern __shared__ float red[];  // [KG][kRows][RT * 16 + 4]
  constexpr int kPitch = RT * 16 + 4;
  pdl_wait();
  pdl_launch_dependents();  // (behind the wait: `expand` reads the plan before its own)
  const int seg = blockIdx.x % p.nseg, ti = blockIdx.x / p.nseg % p.most, split = blockIdx.x / (p.nseg * p.most);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  // head, tile and rows in one round trip (the list has room for every CTA's tile)
  const SmallTile* st = p.small + ti;
  const Tile tile = st->tile;
  const int rows[2] = {st->rows[g], st->rows[8 + g]};
  const int splits = splits_of(p);
  if (!plan_ok(p) || ti >= p.head[p.which] || tile.adapter < 0 || split >= splits) return;
  const int rank = rank_of(p, tile.adapter);
  if (rank == 0) return;
  const Seg& s = p.seg[seg];
  const int steps = (p.K + 31) / 32, ways = splits * KG;
  const int way = split * KG + warp, k0 = (int)((int64_t)way * steps / ways), k1 = (int)((int64_t)(way + 1) * steps / ways);
  const TW* a = static_cast<const TW*>(s.a) + tile.adapter * s.a_adapter + 8 * t;
  const TX* x[NT];
  bool on[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    on[j] = j * 8 + g < tile.count;
    x[j] = static_cast<const TX*>(p.x) + (on[j] ? rows[j] * p.x_row : 0) + 8 * t;
  }
  float c[NT / JT][RT][JT][4];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int m = 0; m < RT; ++m)
#pragma unroll
      for (int e = 0; e < 4; ++e) c[j / JT][m][j % JT][e] = 0.f;
  const int mts = (rank + 15) / 16, nts = (tile.count + 7) / 8;
#pragma unroll 1
  for (int ks = k0; ks < k1; ++ks) {
    const int k = ks * 32;
    const bool kin = k + 8 * t < p.K;
    uint4 xw[NT / JT][JT][F::kLoads], lo[RT], hi[RT];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int l = 0; l < F::kLoads; ++l) xw[j / JT][j % JT][l] = ld16_x(x[j] + k + 4 * l, kin && on[j]);
#pragma unroll
    for (int m = 0; m < RT; ++m) {
      lo[m] = ld16(a + (int64_t)(m * 16 + g) * s.a_row + k, kin && m < mts && m * 16 + g < p.R);
      hi[m] = ld16(a + (int64_t)(m * 16 + 8 + g) * s.a_row + k, kin && m < mts && m * 16 + 8 + g < p.R);
    }
#pragma unroll
    for (int j = 0; j < NT / JT; ++j)
      if (j * JT < nts) F(xw[j]).add(c[j], lo, hi, mts, nts - j * JT);
  }
  // c[m][j]: weight rows 16 m + g and + 8, rows 8 j + 2 t and + 1
  float* mine = red + warp * kRows * kPitch;
#pragma unroll
  for (int m = 0; m < RT; ++m)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) mine[(j * 8 + 2 * t + (e & 1)) * kPitch + m * 16 + g + (e >> 1) * 8] = c[j / JT][m][j % JT][e];
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

// Prompts: a CTA takes a tile's 128 rows, one projection and one of `splits` stretches of K. x and the weights come
// through a ring in shared memory, 128 bytes of each row of x at a time (64 elements, 32 of fp32), which keeps 16 KB a
// stage under way: with operands loaded as above a step waits out the memory's latency (6007 rows of 5120 in bf16:
// 39 us, 26 so). The MMAs' rate is not what bounds it: 8 us of it there.
//
// Warp (rg, kg) has NT x 8 of the rows and, of two, one 32-wide step of a stage. A word lies at its place ^ f(row), f
// such that the lanes that read together, four words of two neighbouring rows, meet no bank twice.
template <typename TX, typename TW, int RT>
struct Long {
  static constexpr int NT = RT <= 4 && !std::is_same_v<TX, float> ? 4 : 2;
  static constexpr int RG = kLarge / (NT * 8), KG = kThreads / 32 / RG;
  static constexpr int MB = RT < 2 ? RT : 2;
  static constexpr int kStep = 128 / (int)sizeof(TX), kSteps = kStep / 32;  // elements of a stage; 32-wide steps
  static constexpr int kXBytes = kLarge * 128, kARow = kStep * 2, kABytes = RT * 16 * kARow;
  static constexpr int kStage = kXBytes + kABytes, kStages = RT == 8 ? 3 : 4;
  static constexpr int kPitch = RT * 16 + 4, kRed = KG * kLarge * kPitch * 4;
  static constexpr int kSmem = kStages * kStage > kRed ? kStages * kStage : kRed;
};
__device__ __forceinline__ int spread(int row) { return ((row & 1) << 2) | ((row >> 1) & 3); }
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool on) {  // zeros where not on
  asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}

template <typename TX, typename TW, int RT>
__global__ void __launch_bounds__(kThreads, RT == 8 && std::is_same_v<TX, float> ? 1 : 2)
    adapter_shrink_long_kernel(const __grid_constant__ Params p) {
  using L = Long<TX, TW, RT>;
  using F = XTerms<TX, TW, L::NT>;
  constexpr int NT = L::NT, KG = L::KG, kPer = 16 / (int)sizeof(TX);  // elements of x in a 16-byte word
  extern __shared__ __align__(128) uint8_t smem[];
  pdl_wait();
  pdl_launch_dependents();  // (behind the wait: the grids behind this one read the plan before their own)
  if (!plan_ok(p)) return;
  const int tiles = min(p.head[p.which], p.most), splits = long_splits(p);
  if ((int)blockIdx.x >= tiles * splits * p.nseg) return;
  const int seg = blockIdx.x % p.nseg, ti = blockIdx.x / p.nseg % tiles, split = blockIdx.x / (p.nseg * tiles);
  const Tile tile = p.tiles[ti];
  if (tile.adapter < 0) return;
  const int rank = rank_of(p, tile.adapter);
  if (rank == 0) return;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int rg = warp % L::RG, kg = warp / L::RG;
  const Seg& s = p.seg[seg];
  const int all = (p.K + L::kStep - 1) / L::kStep;
  const int s0 = (int)((int64_t)split * all / splits), s1 = (int)((int64_t)(split + 1) * all / splits);
  const int mts = (rank + 15) / 16;
  const uint32_t sbase = smem_u32(smem);
  // this thread's words of a stage: word tid % 8 of the rows tid / 8 + 32 i of x, and some of the weights
  int from[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) from[i] = tid / 8 + 32 * i < tile.count ? p.order[tile.begin + tid / 8 + 32 * i] : -1;
  const TW* a = static_cast<const TW*>(s.a) + tile.adapter * s.a_adapter;
  constexpr int kAWords = L::kARow / 16;  // of a row of the weights
  const int arows = min(mts * 16, p.R);
  auto load = [&](int st) {
    if (st < s1) {
      const int k0 = st * L::kStep;
      const uint32_t to = sbase + (st - s0) % L::kStages * L::kStage;
      const int k = k0 + tid % 8 * kPer;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = tid / 8 + 32 * i;
        const bool there = from[i] >= 0 && k < p.K;
        cp_async16(to + r * 128 + ((tid % 8 ^ spread(r)) << 4),
                   static_cast<const TX*>(p.x) + (there ? from[i] * p.x_row + k : 0), there);
      }
#pragma unroll
      for (int w = tid; w < RT * 16 * kAWords; w += kThreads) {
        const int r = w / kAWords, c = w % kAWords;
        const bool there = r < arows && k0 + c * 8 < p.K;
        cp_async16(to + L::kXBytes + r * L::kARow + ((kAWords == 8 ? c ^ spread(r) : c) << 4),
                   there ? a + (int64_t)r * s.a_row + k0 + c * 8 : a, there);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  float c[RT / L::MB][L::MB][NT][4];
#pragma unroll
  for (int m = 0; m < RT; ++m)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) c[m / L::MB][m % L::MB][j][e] = 0.f;
#pragma unroll
  for (int i = 0; i < L::kStages - 1; ++i) load(s0 + i);
#pragma unroll 1
  for (int st = s0; st < s1; ++st) {
    asm volatile("cp.async.wait_group %0;" ::"n"(L::kStages - 2) : "memory");
    __syncthreads();  // this stage is there for all, and the one before it has been read by all
    load(st + L::kStages - 1);
    const uint8_t* xs = smem + (st - s0) % L::kStages * L::kStage;
    const uint8_t* as = xs + L::kXBytes;
    if (rg * NT * 8 >= tile.count) continue;
#pragma unroll
    for (int h = 0; h < L::kSteps; ++h) {
      if (KG > 1 && h != kg) continue;
      uint4 xw[NT][F::kLoads];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const int r = (rg * NT + j) * 8 + g;
#pragma unroll
        for (int l = 0; l < F::kLoads; ++l) {
          const int w = F::kF32 ? 2 * t + l : 4 * h + t;
          xw[j][l] = *reinterpret_cast<const uint4*>(xs + r * 128 + ((w ^ spread(r)) << 4));
        }
      }
      const F terms(xw);
      // (two of the weights' 16 rows at a time: all of them at once leave no registers for a second CTA)
#pragma unroll
      for (int m0 = 0; m0 < RT; m0 += L::MB) {
        if (m0 >= mts) break;
        uint4 lo[L::MB], hi[L::MB];
#pragma unroll
        for (int m = 0; m < L::MB; ++m) {
          const int r = (m0 + m) * 16 + g, w = kAWords == 8 ? 4 * h + t : t;
          lo[m] = *reinterpret_cast<const uint4*>(as + r * L::kARow + ((kAWords == 8 ? w ^ spread(r) : w) << 4));
          hi[m] = *reinterpret_cast<const uint4*>(as + (r + 8) * L::kARow + ((kAWords == 8 ? w ^ spread(r) : w) << 4));
        }
        terms.add(c[m0 / L::MB], lo, hi, mts - m0, NT);
        if (RT > L::MB) asm volatile("" ::: "memory");
      }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  // c[m][j]: weight rows 16 m + g and + 8, rows 8 j + 2 t and + 1 of the warp's
  float* red = reinterpret_cast<float*>(smem);
  float* mine = red + (kg * kLarge + rg * NT * 8) * L::kPitch;
#pragma unroll
  for (int m = 0; m < RT; ++m)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) mine[(j * 8 + 2 * t + (e & 1)) * L::kPitch + m * 16 + g + (e >> 1) * 8] = c[m / L::MB][m % L::MB][j][e];
  __syncthreads();
  const int quads = p.R / 4, live = min((rank + 3) / 4, quads);
  float* h = p.h + ((int64_t)(split * p.nseg + seg) * p.T + tile.begin) * p.R;
  for (int i = tid; i < tile.count * quads; i += kThreads) {
    const int r = i / quads, q = i % quads;
    if (q >= live) continue;
    float4 v = *reinterpret_cast<const float4*>(red + r * L::kPitch + q * 4);
    if constexpr (KG > 1) {
      const float4 u = *reinterpret_cast<const float4*>(red + (kLarge + r) * L::kPitch + q * 4);
      v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
    }
    *reinterpret_cast<float4*>(h + (int64_t)r * p.R + q * 4) = v;
  }
}

// ------------------------------------------------------------------ expand
// Few rows: a CTA takes a tile's 16 rows and a stretch of the outputs of all projections, 32 at a time per warp. h's
// terms lie in shared memory as the MMA's A operands, 16 bytes a lane; the weights are its 8-wide side, with the rows of
// B so assigned that a lane ends up with 8 consecutive outputs of a row. (Prompts: adapters_tc.cu.)
template <typename TW, typename TY, int kBlocks>  // k32 blocks of R at most
__global__ void __launch_bounds__(kExpand, kBlocks == 4 ? 5 : 6) adapter_expand_kernel(const __grid_constant__ Params p) {
  constexpr bool kHalf = std::is_same_v<TW, __half>, kY32 = std::is_same_v<TY, float>;
  constexpr int kTerms = !kHalf && kY32 ? 3 : 2;
  constexpr int kRows = kSmall;
  constexpr int kYWords = 8 * (int)sizeof(TY) / 16;  // 16-byte words of a lane's 8 outputs
  extern __shared__ uint4 frag[];  // [k32 blocks][2][terms][32]
  __shared__ float mul[kRows];
  // The plan, the weights and base were complete before `shrink` let this grid start.
  // (A grid may only end after the one before it, or the one behind it starts too early: every way out waits.)
  pdl_launch_dependents();
  const int range = blockIdx.x % p.ranges, place = blockIdx.x / p.ranges;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const SmallTile* st = p.small + place;  // (read at once, as above)
  Tile tile = st->tile;
  int row[2] = {st->rows[g], st->rows[8 + g]};
  // places without a tile of their own share the others' ranges (72 rows of 18 requests among 64 adapters, rank 104, to
  // 12514 outputs: 60 us without, 40 so)
  const int tiles = max(1, min(p.head[p.which], p.most)), share = p.most / tiles, part = place / tiles;
  if (!plan_ok(p) || part >= share) {
    pdl_wait();
    return;
  }
  if (part > 0) {
    st = p.small + place % tiles;
    tile = st->tile, row[0] = st->rows[g], row[1] = st->rows[8 + g];
  }
  const int rank = tile.adapter < 0 ? 0 : rank_of(p, tile.adapter);
  const int blocks = (rank + 31) / 32;
  // the CTA's pieces, of all projections in a line
  auto pieces = [&](int i) { return (p.seg[i].N + kExpand - 1) / kExpand; };
  int total = 0;
  for (int i = 0; i < p.nseg; ++i) total += pieces(i);
  int first = (int)((int64_t)range * total / p.ranges), last = (int)((int64_t)(range + 1) * total / p.ranges);
  if (share > 1) {
    const int all = last - first;
    last = first + (int)((int64_t)(part + 1) * all / share), first += (int)((int64_t)part * all / share);
  }
#pragma unroll
  for (int e = 0; e < 2; ++e)
    if (e * 8 + g >= tile.count) row[e] = -1;
  const bool copy = rank == 0;
  // A piece's projection, the warp's first output of it, and what of it does not depend on h: the weights of the first
  // k32 block and base.
  struct Piece {
    int seg, n0;
    bool vec;
    uint4 wb[4], bv[2][kYWords];
  };
  auto load_b = [&](const Piece& q, uint4 (&w)[4], int kb) {
    const Seg& s = p.seg[q.seg];
    const TW* b = static_cast<const TW*>(s.b) + (copy ? 0 : tile.adapter * s.b_adapter) + 8 * t;
    const int k = kb * 32 + 8 * t, valid = rank - k;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = q.n0 + 8 * (g >> 1) + 2 * j + (g & 1);
      w[j] = ld16(b + (int64_t)n * s.b_row + kb * 32, valid > 0 && n < s.N);
      if (valid > 0 && valid < 8) {  // columns behind the adapter's rank may hold anything
        uint32_t v[4] = {w[j].x, w[j].y, w[j].z, w[j].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] &= valid >= 2 * i + 2 ? 0xffffffffu : valid == 2 * i + 1 ? 0xffffu : 0u;
        w[j] = make_uint4(v[0], v[1], v[2], v[3]);
      }
    }
  };
  auto fetch = [&](Piece& q, int piece) {
    if (piece >= last) return;
    q.seg = 0;
    for (int k; piece >= (k = pieces(q.seg)); ++q.seg) piece -= k;
    const Seg& s = p.seg[q.seg];
    q.n0 = piece * kExpand + warp * 32;
    load_b(q, q.wb, 0);
    const int n8 = q.n0 + 8 * t;  // the lane's outputs
    q.vec = s.vec && n8 + 8 <= s.N;
    if (!s.base) return;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const TY* from = static_cast<const TY*>(s.base) + (row[e] >= 0 ? row[e] : 0) * s.base_row + n8;
      if (q.vec) {
#pragma unroll
        for (int w = 0; w < kYWords; ++w)
          q.bv[e][w] = row[e] >= 0 ? *(reinterpret_cast<const uint4*>(from) + w) : make_uint4(0, 0, 0, 0);
      } else {  // rows that begin anywhere, and odd ends: an element at a time, all of them under way
        constexpr int kPer = 4 / (int)sizeof(TY);
        uint32_t v[8 / kPer];
#pragma unroll
        for (int i = 0; i < 8 / kPer; ++i) {
          v[i] = 0;
#pragma unroll
          for (int k = 0; k < kPer; ++k)
            if (row[e] >= 0 && n8 + i * kPer + k < s.N) v[i] |= (uint32_t)bits(from[i * kPer + k]) << (16 * k);
        }
#pragma unroll
        for (int w = 0; w < kYWords; ++w) q.bv[e][w] = make_uint4(v[4 * w], v[4 * w + 1], v[4 * w + 2], v[4 * w + 3]);
      }
    }
  };
  int have = -1;  // the projection whose h lies in shared memory
  Piece now, next;
  fetch(now, first);
  pdl_wait();
  for (int piece = first; piece < last; ++piece, now = next) {
    fetch(next, piece + 1);
    const int seg = now.seg;
    const Seg& s = p.seg[seg];
    if (copy && s.base == s.y && s.base_row == s.y_row) continue;  // in place: stays
    if (have != seg && !copy) {
      __syncthreads();  // nobody reads the one before any more
      have = seg;
      // four threads a row: each the words that the lane of its place takes, of every k32 block
      const int r = threadIdx.x >> 2, l = threadIdx.x & 3;
      const bool there = r < tile.count;
      const float* h = p.h + ((int64_t)seg * p.T + tile.begin + r) * p.R + l * 8;
      const int64_t stretch = (int64_t)p.nseg * p.T * p.R;
      const int splits = splits_of(p);  // (here: one register less all along)
      float v[kBlocks][8];
#pragma unroll
      for (int kb = 0; kb < kBlocks; ++kb)
#pragma unroll
        for (int i = 0; i < 8; ++i) v[kb][i] = 0.f;
#pragma unroll (8 / kBlocks)
      for (int q = 0; q < splits; ++q, h += stretch) {
#pragma unroll
        for (int kb = 0; kb < kBlocks; ++kb) {
          if (!there || kb * 32 + l * 8 >= rank) continue;
          const float4 v0 = ld_cg(h + kb * 32), v1 = ld_cg(h + kb * 32 + 4);
          v[kb][0] += v0.x, v[kb][1] += v0.y, v[kb][2] += v0.z, v[kb][3] += v0.w;
          v[kb][4] += v1.x, v[kb][5] += v1.y, v[kb][6] += v1.z, v[kb][7] += v1.w;
        }
      }
      float f = 1.f, back = p.scales ? p.scales[tile.adapter] : 1.f, m = 0.f;
#pragma unroll
      for (int kb = 0; kb < kBlocks; ++kb)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (kb * 32 + l * 8 + i >= rank) v[kb][i] = 0.f;
          m = fmaxf(m, fabsf(v[kb][i]));
        }
      if constexpr (kHalf) {  // the row over a power of two: its largest in [2^14, 2^15)
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
        const int e = (__float_as_int(m) >> 23) - 127;  // 0, denormal and infinite rows stay as they are
        if (e >= -112 && e < 128) f = __int_as_float((14 - e + 127) << 23), back *= __int_as_float((e - 14 + 127) << 23);
      }
      if (l == 0) mul[r] = back;
#pragma unroll
      for (int kb = 0; kb < kBlocks; ++kb) {
        if (kb >= blocks) break;
        // row r of its 16: g = r % 8, words 0 and 2 (r < 8) or 1 and 3
        uint32_t* to = reinterpret_cast<uint32_t*>(frag + kb * 2 * kTerms * 32 + (r & 7) * 4 + l) + (r >> 3);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float v0 = v[kb][2 * i] * f, v1 = v[kb][2 * i + 1] * f;
#pragma unroll
          for (int e = 0; e < kTerms; ++e) {
            const uint32_t w = !kHalf && e == 0 ? pack2<TW>(in_bf16(v0), in_bf16(v1)) : pack2<TW>(v0, v1);
            to[(((i >> 1) * kTerms + e) * 32) * 4 + (i & 1) * 2] = w;
            const float2 u = unpack2<TW>(w);
            v0 = rest(v0, u.x), v1 = rest(v1, u.y);
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
      if (kb + 1 < blocks) load_b(now, wn, kb + 1);
      const uint4* f = frag + (int64_t)kb * 2 * kTerms * 32 + lane;
#pragma unroll
      for (int e = kTerms - 1; e >= 0; --e) {
        const uint4 a0 = f[e * 32], a1 = f[(kTerms + e) * 32];
#pragma unroll
        for (int j = 0; j < 4; ++j) mma16<TW>(c[j], a0.x, a0.y, a0.z, a0.w, now.wb[j].x, now.wb[j].y);
#pragma unroll
        for (int j = 0; j < 4; ++j) mma16<TW>(c[j], a1.x, a1.y, a1.z, a1.w, now.wb[j].z, now.wb[j].w);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) now.wb[j] = wn[j];
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      if (row[e] < 0) continue;
      const float f = copy ? 0.f : mul[e * 8 + g];
      float v[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[2 * j] = c[j][2 * e] * f, v[2 * j + 1] = c[j][2 * e + 1] * f;
      TY* y = static_cast<TY*>(s.y) + row[e] * s.y_row + now.n0 + 8 * t;
      if (s.base) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (kY32) {
            const uint4 w = now.bv[e][i >> 1];
            v[2 * i] += __uint_as_float(i & 1 ? w.z : w.x), v[2 * i + 1] += __uint_as_float(i & 1 ? w.w : w.y);
          } else {
            const uint4 w = now.bv[e][0];
            const float2 q = unpack2<TY>(i == 0 ? w.x : i == 1 ? w.y : i == 2 ? w.z : w.w);
            v[2 * i] += q.x, v[2 * i + 1] += q.y;
          }
        }
      }
      if (now.vec) {
        if constexpr (kY32) {
          reinterpret_cast<float4*>(y)[0] = make_float4(v[0], v[1], v[2], v[3]);
          reinterpret_cast<float4*>(y)[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
          *reinterpret_cast<uint4*>(y) = make_uint4(pack2<TY>(v[0], v[1]), pack2<TY>(v[2], v[3]), pack2<TY>(v[4], v[5]),
                                                    pack2<TY>(v[6], v[7]));
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (now.n0 + 8 * t + i < s.N) y[i] = from_f32<TY>(v[i]);
      }
    }
  }
}

// ------------------------------------------------------------------ launches
bool sizes_ok(int T, int K, int R, int nseg, int n) {
  return T >= 0 && T <= BTF_ADAPTERS_MAX_ROWS && K >= 8 && K % 8 == 0 && K <= (1 << 24) && R >= 8 && R % 8 == 0 &&
         R <= BTF_ADAPTERS_MAX_RANK && nseg >= 1 && nseg <= 3 && n >= 1 && n <= BTF_ADAPTERS_MAX;
}

// Tiles of 16 rows while the rows are few, of 128 for prompts: us as few and as prompts, with the rows of 1 request, of 8
// and each with an adapter of its own. bf16 to 17408, rank 64: 384 rows 21, 27, 28 and 25, 33, 36; 512 rows 33, 31, 41 and
// 25, 30, 37; 1024 rows 52, 67, 69 and 31, 40, 42. fp16 to 4091, rank 24: 512 rows 19, 18, 19 and 28, 28, 38; 1024 rows 37,
// 37, 34 and 30, 41, 40. fp32 q, k and v, whose terms cost the more the fewer rows share their weights: 512 rows 31, 42, 46
// and 38, 47, 95; 1024 rows 60, 70, 75 and 44, 68, 99; 2048 rows 121, 143, 134 and 68, 104, 127.
struct Shape {
  bool large;
  int tiles;   // at most
  int splits;  // stretches of K, at most
};
Shape shape_of(const DeviceInfo& d, int T, int K, int nseg, int n, bool x32) {
  Shape s;
  s.large = T > (x32 ? 1024 : 512);
  const int rows = s.large ? kLarge : kSmall;
  s.tiles = T / rows + std::min(n + 1, T);
  const int least = s.large ? 512 : 256;  // of K that a stretch has
  // for prompts up to kTurns turns of the least tiles, for the small tiles' grid, whose CTAs know their place before they
  // know the plan, at most three quarters of them idle
  const int room = 2 * d.sm_count, least_tiles = (T + rows - 1) / rows;
  s.splits = std::min({s.large ? kTurns * room / (least_tiles * nseg) : std::min(room / (least_tiles * nseg), 4 * room / (s.tiles * nseg)),
                       kMaxSplits, (K + least - 1) / least});
  s.splits = std::max(1, s.splits);
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

template <typename TX, typename TW, int RT>
cudaError_t shrink_rt(const Params& p, bool large, int tiles, cudaStream_t st, bool setup) {
  constexpr int smem = kThreads / 32 * kSmall * (RT * 16 + 4) * 4, smem_long = Long<TX, TW, RT>::kSmem;
  static_assert(Long<TX, TW, RT>::KG <= 2 && smem_long <= 113 * 1024);
  if (setup) {
    if (cudaError_t e = cudaFuncSetAttribute(adapter_shrink_kernel<TX, TW, RT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem))
      return e;
    return cudaFuncSetAttribute(adapter_shrink_long_kernel<TX, TW, RT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_long);
  }
  // what splits_of can come to; CTAs beyond what it takes end at once
  const int most = tiles * p.nseg;
  const dim3 grid((unsigned)(large ? std::max(most, std::min(kTurns * p.room, most * p.splits)) : most * p.splits));
  return large ? launch_pdl(adapter_shrink_long_kernel<TX, TW, RT>, grid, dim3(kThreads), (size_t)smem_long, st, p)
               : launch_pdl(adapter_shrink_kernel<TX, TW, RT>, grid, dim3(kThreads), (size_t)smem, st, p);
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
  // as many pieces each as make about one wave of CTAs
  const int64_t per = std::max<int64_t>(1, (pieces * tiles + 8 * sms - 1) / (8 * sms));
  p.ranges = (int)((pieces + per - 1) / per);
  const dim3 grid((unsigned)(tiles * p.ranges));
  const size_t smem = (size_t)(p.R + 31) / 32 * 2 * terms * 512;
  return p.R <= 32   ? launch_pdl(adapter_expand_kernel<TW, TY, 1>, grid, dim3(kExpand), smem, st, p)
         : p.R <= 64 ? launch_pdl(adapter_expand_kernel<TW, TY, 2>, grid, dim3(kExpand), smem, st, p)
                     : launch_pdl(adapter_expand_kernel<TW, TY, 4>, grid, dim3(kExpand), smem, st, p);
}

}  // namespace

int adapters_setup(DeviceInfo& d) {
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
  if (T == 0) return 0;
  int64_t bytes = 0;  // whatever x's type
  for (bool x32 : {false, true}) bytes = std::max(bytes, Work(shape_of(*dev, T, K, nseg, n_adapters, x32), T, R, nseg).bytes);
  return bytes;
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
  // (of one row or adapter no stride matters)
  const int64_t x_row = a->T > 1 ? a->x_row : 0;
  if (!a->x || !a->plan || !al(a->x) || !al(a->plan) || x_row < 0 || x_row * xb % 16)
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
    const int64_t a_adapter = a->n_adapters > 1 ? s.a_adapter : 0, b_adapter = a->n_adapters > 1 ? s.b_adapter : 0;
    const int64_t b_row = s.N > 1 ? s.b_row : 0;
    for (int64_t v : {a_adapter, s.a_row, b_adapter, b_row})
      if (v < 0 || v % 8) return fail(BTF_ERR_ARG, "btf_adapters: the strides of a and b must be multiples of 8 elements, >= 0");
    if (s.a_row == 0 || (s.N > 1 && b_row == 0)) return fail(BTF_ERR_ARG, "btf_adapters: the rows of a and b need a stride");
    if (reinterpret_cast<uintptr_t>(s.y) % yb || reinterpret_cast<uintptr_t>(s.base) % yb)
      return fail(BTF_ERR_ARG, "btf_adapters: y or base is not aligned to its type");
    if (a->T > 1 && s.y_row < s.N) return fail(BTF_ERR_ARG, "btf_adapters: the rows of y overlap");
    if (s.base && a->T > 1 && s.base_row < 0) return fail(BTF_ERR_ARG, "btf_adapters: the stride of base is negative");
    if (s.base == s.y && a->T > 1 && s.base_row != s.y_row)
      return fail(BTF_ERR_ARG, "btf_adapters: in place needs the same strides");
    const int64_t y_row = a->T > 1 ? s.y_row : 0, base_row = a->T > 1 ? s.base_row : 0;
    const bool vec = al(s.y) && y_row * yb % 16 == 0 && al(s.base) && base_row * yb % 16 == 0;
    p.seg[i] = {s.a, s.b, s.base, s.y, a_adapter, s.a_row, b_adapter, b_row, base_row, y_row, s.N, vec};
  }
  const DeviceInfo* dev = current_device();
  if (!dev) return BTF_ERR_STATE;
  const Shape sh = shape_of(*dev, a->T, a->K, a->nseg, a->n_adapters, a->x_type == BTF_F32);
  const Work w(sh, a->T, a->R, a->nseg);
  if (!a->work || !al(a->work) || a->work_bytes < w.bytes)
    return fail(BTF_ERR_ARG, "btf_adapters: workspace null, not 16-byte aligned or too small (%lld bytes, %lld are needed)",
                (long long)a->work_bytes, (long long)w.bytes);
  const PlanLayout at(a->T, a->n_adapters);
  const uint8_t* plan = static_cast<const uint8_t*>(a->plan);
  p.x = a->x, p.x_row = x_row;
  p.T = a->T, p.K = a->K, p.R = a->R, p.n = a->n_adapters, p.nseg = a->nseg, p.splits = sh.splits, p.room = 2 * dev->sm_count, p.most = sh.tiles, p.ranges = 1;
  p.steps = (a->K * elem_bytes(a->x_type) + 127) / 128;
  p.ranks = a->ranks, p.scales = a->scales;
  p.head = reinterpret_cast<const int32_t*>(plan), p.order = reinterpret_cast<const int32_t*>(plan + at.order);
  p.owner = reinterpret_cast<const int32_t*>(plan + at.owner);
  p.tiles = reinterpret_cast<const Tile*>(plan + at.large), p.small = reinterpret_cast<const SmallTile*>(plan + at.small);
  p.which = sh.large ? 3 : 2;
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
