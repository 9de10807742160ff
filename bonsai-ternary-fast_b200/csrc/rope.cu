// Rotary positions (btf_rope): the q and k of T tokens turned by their
// positions, with the optional per-head RMSNorm before it and the conversion to
// the cache's type and row after it, up to three tensors in one launch.
//
//   (a, b) -> m (a cos t - b sin t, a sin t + b cos t),  t = pos * f_i
//
// t in turns is pos * (f_i / 2 pi) in 64 bits: off by |turns| 2^-52 or so (the
// frequency's rounding and the product's). Its fraction is rounded to fp32 (2^-26 of a
// turn), so cos and sin are good to 2^-22 while the former is the smaller, up to 2^26
// turns (positions of 4 10^8 at f = 1); at 2^31 they are off by 2^-24 of a turn, 4e-7,
// more. (pos * f_i in fp32 loses 2^-24 pos radians: 0.06 at 10^6.)
//
// What bounds it: bytes, each read and written once, for prompts and gradients (see
// rope_heads; 7001 tokens of 40 fp32 heads of 80 in 32.2 us, 5.6 TB/s); the launch for
// a few tokens (1 token of 24 + 4 + 4 heads of 256 with norm and append: 3.1 us, 61
// tokens of 32 + 8 + 8 heads of 128: 4.4). So the angles are worked out once per token
// and thread and used for all heads that the thread takes, whole 16-byte words move,
// and q, k and v share a launch.
#include <cmath>
#include <type_traits>

#include "elem.cuh"

namespace btf {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxHeads = 16;  // per thread
// NORM: none; a token's lanes hold a whole head; or they take several rounds for one
constexpr int kOneRound = 1, kRounds = 2;

struct RopeSeg {
  const void* x;
  void* y;
  int64_t x_token, x_head, y_token, y_head, n_rows;
  const float* normw;
  const int32_t* rows;
  int heads;
  uint8_t x_type, y_type, rotate;
  int block0;  // first head block (grid y) of this tensor
};
struct RopeParams {
  RopeSeg seg[3];
  int nseg, T, D, R, inter, inverse;
  int lanes;  // threads per token: its items (with a norm a power of two, at most 32)
  int hl;     // heads per thread
  const double* turns;
  const int32_t* pos;
  float mscale, eps;
  // several axes: each pair's axis, and the elements from one axis's positions to the next's
  const uint8_t* axis;
  int64_t pos_axis;
  int n_axes;
};
// A launch costs the host 0.4 us more from somewhere between 344 and 368 bytes of parameters on (one token: 4.1 and 4.5 us a
// call of the C ABI), more than the rest of this file's host side.
static_assert(sizeof(RopeParams) <= 344);

// 1 / sqrt(mean square + eps) of a head from its lanes' sums of squares.
__device__ __forceinline__ float norm_scale(const RopeParams& p, unsigned mask, float ss) {
  for (int o = p.lanes >> 1; o; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
  return 1.0f / sqrtf(ss / (float)p.D + p.eps);
}

// One token's heads [h0, h1) of one tensor; scales: the token's place for their norms. A thread owns the C pairs of its
// item (and item + lanes, ... when a head has more items than lanes) and keeps
// their cos and sin over the heads. The loads of kBatch heads are issued before
// the first store: x and y may be one tensor, so the compiler would keep each
// head's loads behind the stores of the one before. 16384 tokens of 32 + 8 bf16
// heads of 128, 336 MB: 100 us a head at a time, 67 with 4, 60 with 8, 57 (5870
// GB/s, 0.90 of a plain copy's rate) with 16 heads a thread for 8; loads ahead of
// the angles too keep more registers and lose.
//
// AXES: pair i turns by the token's position on its axis. All positions of the token (at most four) are read at once
// and picked from, so that no read waits for the axis.
template <typename TX, typename TY, int C, int NORM, bool AXES>
__device__ __forceinline__ void rope_heads(const RopeParams& p, const RopeSeg& s, int t, int64_t row, int h0, int h1,
                                           int lane, float* scales) {
  constexpr int kBatch = NORM ? 1 : C == 8 ? 8 : 4;
  const int R = s.rotate ? p.R : 0, half = R / 2, D = p.D;
  const int nrot = half / C;                               // rotated items: C pairs each
  const int items = nrot + (D - R + 2 * C - 1) / (2 * C);  // copied items: 2 C elements each
  const TX* x = static_cast<const TX*>(s.x) + (int64_t)t * s.x_token;
  TY* y = static_cast<TY*>(s.y) + row * s.y_token;
  // with a norm: the lanes of this token, which take the same branches
  const unsigned mask = p.lanes == 32 ? 0xffffffffu : ((1u << p.lanes) - 1) << (threadIdx.x & 31 & ~(p.lanes - 1));
  // in place, a round's stores replace values that the next one's sum would read: every head's scale is taken before
  // the first store (such a token has a warp). Once a head, not once a round: 4000 tokens of 16 fp16 heads of 1024 take
  // 194 us for 357.
  if (NORM == kRounds && s.normw) {
#pragma unroll 1
    for (int h = h0; h < h1; ++h) {
      const TX* xh = x + (int64_t)h * s.x_head;
      float ss = 0.f;
      for (int e = lane; e < D; e += p.lanes) {
        const float v = to_f32(xh[e]);
        ss = fmaf(v, v, ss);
      }
      const float scale = norm_scale(p, mask, ss);
      if (lane == 0) scales[h - h0] = scale;
    }
    __syncwarp(mask);
  }
  for (int it0 = 0; it0 < (NORM == kOneRound ? 1 : items); it0 += p.lanes) {  // rounds
    const int it = it0 + lane;
    const bool active = it < items, rot = it < nrot;
    if (!NORM && !active) return;
    // the item's two chunks of C elements
    const int i = it * C, ca = rot ? (p.inter ? 2 * i : i) : R + (it - nrot) * 2 * C;
    const int cb = rot && !p.inter ? half + i : ca + C;
    const bool hasb = active && cb < D;
    float cs[C], sn[C];
    if (rot) {
      int at[AXES ? BTF_ROPE_MAX_AXES : 1];
      at[0] = p.pos[t];
      if constexpr (AXES) {
#pragma unroll
        for (int a = 1; a < BTF_ROPE_MAX_AXES; ++a) at[a] = a < p.n_axes ? p.pos[a * p.pos_axis + t] : at[0];
      }
#pragma unroll
      for (int j = 0; j < C; ++j) {
        int on = at[0];
        if constexpr (AXES) {
          const int ax = p.axis[i + j];
#pragma unroll
          for (int a = 1; a < BTF_ROPE_MAX_AXES; ++a) on = ax == a ? at[a] : on;
        }
        const double turn = (double)on * p.turns[i + j];
        const float f = (float)(turn - rint(turn));
        float sv, cv;
        sincospif(2.0f * f, &sv, &cv);
        cs[j] = cv * p.mscale;
        sn[j] = p.inverse ? -sv * p.mscale : sv * p.mscale;
      }
    }
    float wa[C], wb[C];
    if (NORM && s.normw) {
#pragma unroll
      for (int j = 0; j < C; ++j) {
        wa[j] = active ? s.normw[ca + j] : 0.f;
        wb[j] = hasb ? s.normw[cb + j] : 0.f;
      }
    }
#pragma unroll 1
    for (int hb = h0; hb < h1; hb += kBatch) {
      Pack<TX, C> a[kBatch] = {}, b[kBatch] = {};
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const TX* xh = x + (int64_t)(hb + k) * s.x_head;
        if (active && hb + k < h1) a[k].load(xh + ca);
        if (hasb && hb + k < h1) b[k].load(xh + cb);
      }
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        if (kBatch > 1 && hb + k >= h1) break;
        float fa[C], fb[C];
#pragma unroll
        for (int j = 0; j < C; ++j) fa[j] = a[k].get(j), fb[j] = b[k].get(j);
        if (NORM && s.normw) {
          float scale;
          if constexpr (NORM == kRounds) {
            scale = scales[hb - h0];
          } else {  // the token's lanes hold the whole head
            float ss = 0.f;
#pragma unroll
            for (int j = 0; j < C; ++j) ss = fmaf(fa[j], fa[j], fmaf(fb[j], fb[j], ss));
            scale = norm_scale(p, mask, ss);
          }
#pragma unroll
          for (int j = 0; j < C; ++j) fa[j] *= scale * wa[j], fb[j] *= scale * wb[j];
        }
        Pack<TY, C> oa, ob;
        if (!rot) {
#pragma unroll
          for (int j = 0; j < C; ++j) oa.set(j, fa[j]), ob.set(j, fb[j]);
        } else if (!p.inter) {
#pragma unroll
          for (int j = 0; j < C; ++j) {
            oa.set(j, fmaf(fa[j], cs[j], -fb[j] * sn[j]));
            ob.set(j, fmaf(fa[j], sn[j], fb[j] * cs[j]));
          }
        } else {
          float v[2 * C];
#pragma unroll
          for (int j = 0; j < C; ++j) v[j] = fa[j], v[C + j] = fb[j];
#pragma unroll
          for (int j = 0; j < C; ++j) {
            const float e = v[2 * j], o = v[2 * j + 1];
            v[2 * j] = fmaf(e, cs[j], -o * sn[j]);
            v[2 * j + 1] = fmaf(e, sn[j], o * cs[j]);
          }
#pragma unroll
          for (int j = 0; j < C; ++j) oa.set(j, v[j]), ob.set(j, v[C + j]);
        }
        TY* yh = y + (int64_t)(hb + k) * s.y_head;
        if (active) oa.store(yh + ca);
        if (hasb) ob.store(yh + cb);
      }
    }
  }
}

template <typename TX, int C, int NORM, bool AXES>
__device__ __forceinline__ void rope_to(const RopeParams& p, const RopeSeg& s, int t, int64_t row, int h0, int h1,
                                        int lane, float* scales) {
  if (s.y_type == BTF_F32) rope_heads<TX, float, C, NORM, AXES>(p, s, t, row, h0, h1, lane, scales);
  else if (s.y_type == BTF_F16) rope_heads<TX, __half, C, NORM, AXES>(p, s, t, row, h0, h1, lane, scales);
  else rope_heads<TX, __nv_bfloat16, C, NORM, AXES>(p, s, t, row, h0, h1, lane, scales);
}

template <int C, int NORM, bool AXES>
__global__ void __launch_bounds__(kThreads) rope_kernel(const __grid_constant__ RopeParams p) {
  __shared__ float scales_of[NORM == kRounds ? kThreads / 32 : 1][kMaxHeads];
  float* scales = scales_of[NORM == kRounds ? threadIdx.x >> 5 : 0];
  pdl_launch_dependents();
  pdl_wait();
  const int per = kThreads / p.lanes, in = threadIdx.x / p.lanes;
  const int t = blockIdx.x * per + in, lane = threadIdx.x - in * p.lanes;
  int si = 0;
  while (si + 1 < p.nseg && (int)blockIdx.y >= p.seg[si + 1].block0) ++si;
  const RopeSeg& s = p.seg[si];
  const int h0 = ((int)blockIdx.y - s.block0) * p.hl, h1 = min(h0 + p.hl, s.heads);
  if (in >= per || t >= p.T) return;
  int64_t row = t;
  if (s.rows) {
    row = s.rows[t];
    if (row < 0 || row >= s.n_rows) return;
  }
  if constexpr (C != 8 || NORM)  // the host takes 4 for fp32 without a norm
    if (s.x_type == BTF_F32) return rope_to<float, C, NORM, AXES>(p, s, t, row, h0, h1, lane, scales);
  if (s.x_type == BTF_F16) rope_to<__half, C, NORM, AXES>(p, s, t, row, h0, h1, lane, scales);
  else rope_to<__nv_bfloat16, C, NORM, AXES>(p, s, t, row, h0, h1, lane, scales);
}

bool aligned_for(const btf_rope_seg& s, int C) {
  auto ok = [C](const void* ptr, int type, int64_t a, int64_t b) {
    const int bytes = C * elem_bytes(type), al = bytes < 16 ? bytes : 16;
    return reinterpret_cast<uintptr_t>(ptr) % al == 0 && a * elem_bytes(type) % al == 0 &&
           b * elem_bytes(type) % al == 0;
  };
  return ok(s.x, s.x_type, s.x_token, s.x_head) && ok(s.y, s.y_type, s.y_token, s.y_head);
}

}  // namespace
}  // namespace btf

using namespace btf;

extern "C" {

int btf_rope_table(const btf_rope_cfg* c, double* turns, float* mscale) {
  if (!c || !turns || !mscale) return fail(BTF_ERR_ARG, "btf_rope_table: null argument");
  const int R = c->n_rot;
  if (R < 2 || R % 2 || R > BTF_ROPE_MAX_D)
    return fail(BTF_ERR_ARG, "btf_rope_table: n_rot must be even, 2..%d (got %d)", BTF_ROPE_MAX_D, R);
  if (!(c->base > 1) || !std::isfinite(c->base)) return fail(BTF_ERR_ARG, "btf_rope_table: base must be > 1");
  if (c->scaling < BTF_ROPE_NONE || c->scaling > BTF_ROPE_YARN)
    return fail(BTF_ERR_ARG, "btf_rope_table: unknown scaling %d", c->scaling);
  const double s = c->scaling == BTF_ROPE_NONE ? 1.0 : c->factor;
  if (!(s >= 1) || !std::isfinite(s)) return fail(BTF_ERR_ARG, "btf_rope_table: factor must be >= 1");
  const double two_pi = 6.283185307179586476925286766559;
  double base = c->base, lo = 0, hi = 0;
  if (c->scaling == BTF_ROPE_NTK) {
    if (R < 4) return fail(BTF_ERR_ARG, "btf_rope_table: NTK scaling needs n_rot >= 4");
    base *= std::pow(s, (double)R / (R - 2));
  }
  *mscale = 1.0f;
  if (c->scaling == BTF_ROPE_YARN) {
    if (c->orig_ctx < 1 || !(c->beta_slow > 0) || !(c->beta_fast >= c->beta_slow) || !std::isfinite(c->beta_fast))
      return fail(BTF_ERR_ARG, "btf_rope_table: yarn needs orig_ctx >= 1 and beta_fast >= beta_slow > 0");
    auto d = [&](double b) { return R * std::log(c->orig_ctx / (two_pi * b)) / (2 * std::log(base)); };
    lo = std::max(std::floor(d(c->beta_fast)), 0.0);
    hi = std::min(std::ceil(d(c->beta_slow)), R - 1.0);
    *mscale = (float)(0.1 * std::log(s) + 1.0);
  }
  for (int i = 0; i < R / 2; ++i) {
    double f = std::pow(base, -2.0 * i / R);
    if (c->scaling == BTF_ROPE_LINEAR) f /= s;
    if (c->scaling == BTF_ROPE_YARN) {
      const double r = std::min(1.0, std::max(0.0, (i - lo) / std::max(hi - lo, 0.001)));
      f = f * (1 - r) + f / s * r;
    }
    turns[i] = f / two_pi;
  }
  return BTF_OK;
}

int btf_rope_axes_table(const btf_rope_cfg* c, const int* sections, int n_axes, int layout, double* turns, uint8_t* axis,
                        float* mscale) {
  if (!c || !sections || !turns || !axis || !mscale) return fail(BTF_ERR_ARG, "btf_rope_axes_table: null argument");
  if (n_axes < 1 || n_axes > BTF_ROPE_MAX_AXES)
    return fail(BTF_ERR_ARG, "btf_rope_axes_table: 1..%d axes (got %d)", BTF_ROPE_MAX_AXES, n_axes);
  if (layout < BTF_AXES_SPLIT || layout > BTF_AXES_OWN)
    return fail(BTF_ERR_ARG, "btf_rope_axes_table: unknown layout %d", layout);
  int64_t pairs = 0;
  for (int a = 0; a < n_axes; ++a) {
    if (sections[a] < 0 || sections[a] > BTF_ROPE_MAX_D / 2)
      return fail(BTF_ERR_ARG, "btf_rope_axes_table: an axis has 0..%d pairs (got %d)", BTF_ROPE_MAX_D / 2, sections[a]);
    pairs += sections[a];
  }
  if (2 * pairs != c->n_rot)
    return fail(BTF_ERR_ARG, "btf_rope_axes_table: the axes have %lld pairs, n_rot is %d", (long long)pairs, c->n_rot);
  if (pairs == 0) return fail(BTF_ERR_ARG, "btf_rope_axes_table: the axes have no pairs");
  btf_rope_cfg own = *c;
  if (layout != BTF_AXES_OWN) {
    if (int rc = btf_rope_table(c, turns, mscale)) return rc;
  }
  int left[BTF_ROPE_MAX_AXES], at = 0;
  for (int a = 0; a < n_axes; ++a) {
    left[a] = sections[a];
    if (layout == BTF_AXES_TURNS) continue;
    own.n_rot = 2 * sections[a];
    if (layout == BTF_AXES_OWN && sections[a])
      if (int rc = btf_rope_table(&own, turns + at, mscale)) return rc;
    for (int j = 0; j < sections[a]; ++j) axis[at++] = (uint8_t)a;
  }
  for (int a = 0; at < pairs; a = (a + 1) % n_axes)  // in turn
    if (left[a]) --left[a], axis[at++] = (uint8_t)a;
  return BTF_OK;
}

}  // extern "C"

namespace {

// Both calls; axis NULL: one position per token.
int rope_call(const btf_rope_seg* segs, int nseg, int T, int D, int n_rot, const double* turns, float mscale,
              int interleaved, int inverse, float eps, const int32_t* pos, const uint8_t* axis, int n_axes,
              int64_t pos_axis, void* stream) {
  if (!segs || nseg < 1 || nseg > 3) return fail(BTF_ERR_ARG, "btf_rope: 1..3 tensors (got %d)", nseg);
  if (T < 0 || T > 1 << 30) return fail(BTF_ERR_ARG, "btf_rope: T must be 0..2^30 (got %d)", T);
  if (D < 1 || D > BTF_ROPE_MAX_D || n_rot < 0 || n_rot % 2 || n_rot > D)
    return fail(BTF_ERR_ARG, "btf_rope: need 1 <= D <= %d and an even 0 <= n_rot <= D (got %d, %d)", BTF_ROPE_MAX_D, D,
                n_rot);
  if (T == 0) return BTF_OK;
  RopeParams p{};
  bool rotates = false, norm = false, wide = false;
  int64_t heads = 0;
  int C = 8;
  if (n_rot % 16 || D % 8) C = n_rot % 8 || D % 4 ? 1 : 4;
  for (int i = 0; i < nseg; ++i) {
    const btf_rope_seg& s = segs[i];
    if (s.heads < 0 || s.heads > 65536) return fail(BTF_ERR_ARG, "btf_rope: heads must be 0..65536");
    if (!elem_type_ok(s.x_type) || !elem_type_ok(s.y_type)) return fail(BTF_ERR_ARG, "btf_rope: unknown element type");
    if (s.heads && (!s.x || !s.y)) return fail(BTF_ERR_ARG, "btf_rope: null tensor");
    if (s.heads && (reinterpret_cast<uintptr_t>(s.x) % elem_bytes(s.x_type) ||
                    reinterpret_cast<uintptr_t>(s.y) % elem_bytes(s.y_type)))
      return fail(BTF_ERR_ARG, "btf_rope: a tensor is not aligned to its type");
    if (s.heads && ((s.heads > 1 && s.y_head == 0) || (T > 1 && s.y_token == 0 && !(s.rows && s.n_rows == 1))))
      return fail(BTF_ERR_ARG, "btf_rope: the heads and rows of y need strides");
    if (s.normw && inverse) return fail(BTF_ERR_ARG, "btf_rope: the inverse has no norm");
    if (s.rows && s.n_rows < 1) return fail(BTF_ERR_ARG, "btf_rope: rows without n_rows");
    if (s.heads && s.x == s.y &&
        (s.x_type != s.y_type || s.rows || s.x_token != s.y_token || s.x_head != s.y_head))
      return fail(BTF_ERR_ARG, "btf_rope: in place needs one type, the same strides and no rows");
    rotates |= s.heads > 0 && s.rotate && n_rot > 0;
    norm |= s.heads && s.normw;
    wide |= s.heads && s.x_type == BTF_F32;
    heads += s.heads;
    if (C == 8 && !aligned_for(s, 8)) C = 4;
    if (C == 4 && !aligned_for(s, 4)) C = 1;
  }
  if (rotates && (!turns || !pos)) return fail(BTF_ERR_ARG, "btf_rope: null turns or pos");
  if (heads == 0) return BTF_OK;
  const DeviceInfo* dev = current_device();
  if (!dev) return BTF_ERR_STATE;
  p.nseg = 0;
  p.T = T, p.D = D, p.R = n_rot, p.inter = interleaved != 0, p.inverse = inverse != 0;
  p.turns = turns, p.pos = pos, p.mscale = mscale, p.eps = eps;
  p.axis = axis, p.n_axes = n_axes, p.pos_axis = pos_axis;
  // fp32 without a norm: 4 pairs an item, one 16-byte word a load and twice the threads (16384 tokens of
  // 16 + 16 interleaved heads of 80: 59 us, 76 with 8 pairs, whose words lie 32 bytes apart from lane to lane)
  if (C == 8 && !norm && wide) C = 4;
  const int items = std::max(n_rot / 2 / C + (D - n_rot + 2 * C - 1) / (2 * C), (D + 2 * C - 1) / (2 * C));
  // with a norm a token's lanes sum over a head by shuffles: a power of two of them
  p.lanes = norm ? 1 : std::min(items, kThreads);
  while (norm && p.lanes < items && p.lanes < 32) p.lanes *= 2;
  // heads per thread: more of them share one cos and sin, as long as the card
  // stays full; 16 pay where 8 are in flight at once (7001 tokens of 40 fp32 heads
  // of 80: 32.5 us with 8, 34.7 with 16)
  const int64_t full = (int64_t)dev->sm_count * 2048;
  p.hl = (int)std::max<int64_t>(1, std::min<int64_t>(C == 8 && !wide ? kMaxHeads : 8, (int64_t)T * heads * p.lanes / full));
  int blocks = 0;
  for (int i = 0; i < nseg; ++i) {
    const btf_rope_seg& s = segs[i];
    if (s.heads == 0) continue;
    p.seg[p.nseg++] = {s.x, s.y, s.x_token, s.x_head, s.y_token, s.y_head, s.n_rows, s.normw, s.rows, s.heads,
                       (uint8_t)s.x_type, (uint8_t)s.y_type, (uint8_t)(s.rotate != 0 && n_rot > 0), blocks};
    blocks += (s.heads + p.hl - 1) / p.hl;
  }
  if (blocks > 65535) return fail(BTF_ERR_UNSUPPORTED, "btf_rope: too many heads for one launch");
  const int per = kThreads / p.lanes;
  const dim3 grid((T + per - 1) / per, blocks);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const auto pick = [C](auto c8, auto c4, auto c1) { return C == 8 ? c8 : C == 4 ? c4 : c1; };
  const auto kernel_of = [&](auto axes) {
    constexpr bool A = decltype(axes)::value;
    return !norm             ? pick(rope_kernel<8, 0, A>, rope_kernel<4, 0, A>, rope_kernel<1, 0, A>)
           : items > p.lanes ? pick(rope_kernel<8, kRounds, A>, rope_kernel<4, kRounds, A>, rope_kernel<1, kRounds, A>)
                             : pick(rope_kernel<8, kOneRound, A>, rope_kernel<4, kOneRound, A>, rope_kernel<1, kOneRound, A>);
  };
  const auto kernel = axis ? kernel_of(std::true_type{}) : kernel_of(std::false_type{});
  const cudaError_t e = launch_pdl(kernel, grid, dim3(kThreads), 0, st, p);
  return e == cudaSuccess ? BTF_OK : cuda_fail(e, "btf_rope");
}

}  // namespace

extern "C" {

int btf_rope(const btf_rope_seg* segs, int nseg, int T, int D, int n_rot, const double* turns, float mscale,
             int interleaved, int inverse, float eps, const int32_t* pos, void* stream) {
  return rope_call(segs, nseg, T, D, n_rot, turns, mscale, interleaved, inverse, eps, pos, nullptr, 1, 0, stream);
}

int btf_rope_axes(const btf_rope_seg* segs, int nseg, int T, int D, int n_rot, const double* turns, const uint8_t* axis,
                  int n_axes, float mscale, int interleaved, int inverse, float eps, const int32_t* pos,
                  int64_t pos_axis, void* stream) {
  if (n_axes < 1 || n_axes > BTF_ROPE_MAX_AXES)
    return fail(BTF_ERR_ARG, "btf_rope_axes: 1..%d axes (got %d)", BTF_ROPE_MAX_AXES, n_axes);
  if (n_rot > 0 && T > 0 && !axis) return fail(BTF_ERR_ARG, "btf_rope_axes: null axis");
  if (n_axes > 1 && pos_axis < 0) return fail(BTF_ERR_ARG, "btf_rope_axes: the stride between the axes' positions is negative");
  return rope_call(segs, nseg, T, D, n_rot, turns, mscale, interleaved, inverse, eps, pos, n_rot > 0 ? axis : nullptr,
                   n_axes, pos_axis, stream);
}

}  // extern "C"
