// Shared by the two halves of the low-rank adapters: few rows (adapters.cu) and
// prompts on tcgen05 (adapters_tc.cu).
#pragma once
#include <algorithm>
#include <climits>

#include "elem.cuh"

namespace btf {
namespace adapt {

constexpr int kSmall = 16, kLarge = 128;  // rows of a tile
constexpr int kMaxSplits = 16;
constexpr int kTurns = 4;
constexpr int kItemSteps = 5;  // what an item costs beside its steps: the ring's filling, h
constexpr int kErrPlan = 2;  // device error word: a plan of other sizes

struct Tile {
  int adapter, begin, count, unused;  // adapter -1: rows without one
};
struct SmallTile {
  Tile tile;
  int32_t rows[kSmall];  // the first `count` of them
};
// The plan in memory: 8 words {T, adapters, small tiles, large tiles, rows with an
// adapter}, the rows in order, the adapter of each (n: none), then both lists of tiles.
struct PlanLayout {
  int64_t order, owner, small, large, bytes;
  PlanLayout(int64_t T, int64_t n) {
    const int64_t lists = std::min(n + 1, T) + 1;
    order = 32;
    owner = order + 4 * T;
    small = (owner + 4 * T + 15) / 16 * 16;
    large = small + (int64_t)sizeof(SmallTile) * (T / kSmall + lists);
    bytes = large + (int64_t)sizeof(Tile) * (T / kLarge + lists);
  }
};

struct Seg {
  const void *a, *b, *base;
  void* y;
  int64_t a_adapter, a_row, b_adapter, b_row, base_row, y_row;
  int N;
  int vec;  // y (and base) take whole 16-byte words
};
struct Params {
  Seg seg[3];
  const void* x;
  int64_t x_row;
  int T, K, R, n, nseg, ranges;
  int splits, room;  // stretches of K at most; CTAs that they may come to
  int most, steps;   // tiles at most; steps of K (prompts)
  const int32_t* ranks;
  const float* scales;
  const int32_t *head, *order, *owner;
  const Tile* tiles;  // the large ones
  const SmallTile* small;
  int which;  // the plan's word with the number of tiles
  float* h;   // [splits][nseg][T][R]
  // prompts: h as the MMAs take it, [terms][nseg][T][R to whole 64], and each row's factor [nseg][T]
  uint16_t* terms;
  float* mul;
  int* err;
};

__device__ __forceinline__ bool plan_ok(const Params& p) {
  if (p.head[0] == p.T && p.head[1] == p.n) return true;
  if (blockIdx.x == 0 && threadIdx.x == 0) atomicCAS(p.err, 0, kErrPlan);
  return false;
}
__device__ __forceinline__ int rank_of(const Params& p, int a) { return p.ranks ? min(max(p.ranks[a], 0), p.R) : p.R; }
// The stretches of K, by the tiles that there are: 256 rows of one request among 24 adapters are 16 tiles, where up to 41
// could be (256 fp32 rows, q, k and v: 29 us with the stretches that room for all of them leaves, 23 so).
__device__ __forceinline__ int splits_of(const Params& p) {
  return max(1, min(p.splits, p.room / (min(max(p.head[p.which], 1), p.most) * p.nseg)));
}
// The same for prompts, by how many turns of how many steps the CTAs then take (whole warps; 6007 fp32 rows of 8
// requests, 156 items for 296 places: 375 us in one turn, 254 so; 1024 rows of one, 24 items: 114 and 46).
__device__ __forceinline__ int long_splits(const Params& p) {
  const int items = min(max(p.head[p.which], 1), p.most) * p.nseg, s = (threadIdx.x & 31) + 1;
  const int turns = (items * s + p.room - 1) / p.room, each = (p.steps + s - 1) / s + kItemSteps;
  const int cost = s == 1 || (s <= p.splits && turns <= kTurns) ? turns * each : INT_MAX;
  return __ffs(__ballot_sync(0xffffffffu, cost == __reduce_min_sync(0xffffffffu, cost)));
}

// What `shrink` wrote: never from L1, and in its place behind the wait.
__device__ __forceinline__ float4 ld_cg(const float* p) {
  float4 v;
  asm volatile("ld.global.cg.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p) : "memory");
  return v;
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (std::is_same_v<T, __half>) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (std::is_same_v<T, __half>) {
    const __half2 h = *reinterpret_cast<const __half2*>(&w);
    return __half22float2(h);
  } else {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
}
__device__ __forceinline__ uint32_t bits(float v) { return __float_as_uint(v); }
__device__ __forceinline__ uint32_t bits(__half v) { return __half_as_ushort(v); }
__device__ __forceinline__ uint32_t bits(__nv_bfloat16 v) { return __bfloat16_as_ushort(v); }
// v for its first bf16 term: a finite v rounds to a finite one (the next term has the rest, and all of an infinity or NaN)
__device__ __forceinline__ float in_bf16(float v) { return fminf(fmaxf(v, -0x1.fep127f), 0x1.fep127f); }
// What is left of v behind its first term (0 behind an infinity, not inf - inf).
__device__ __forceinline__ float rest(float v, float term) { return v == term ? 0.f : v - term; }

}  // namespace adapt
}  // namespace btf
