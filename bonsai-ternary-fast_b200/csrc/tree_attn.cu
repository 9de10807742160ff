// Attention for a tree of drafted tokens over a cache (btf_tree_attention).
#include <algorithm>
#include <cmath>

#include "elem.cuh"

namespace btf {
namespace {

constexpr int kWarps = 8;

struct TreeParams {
  const void *q, *k, *v;
  void* o;
  int64_t q_batch, q_node, q_head, kv_batch, kv_row, kv_head, o_batch, o_node, o_head;
  int n, H, HK, D, n_ctx;
  const int32_t *lens, *parents, *counts;
  float scale;
};

// Itself and its ancestors, as bits, for the n nodes of a tree: pointer doubling
// over the parents (a parent that is not an earlier node hangs on the cache).
// One warp, two nodes per lane; masks go to `out`.
__device__ __forceinline__ void tree_masks(const int32_t* parents, int n, uint64_t* out, int* jump) {
  const int lane = threadIdx.x & 31;
  for (int j = lane; j < 64; j += 32) {
    const int pj = j < n ? parents[j] : -1;
    jump[j] = pj >= 0 && pj < j ? pj : -1;
    out[j] = 1ull << j;
  }
  __syncwarp();
  for (int s = 0; s < 6; ++s) {
    uint64_t m[2];
    int jj[2];
    for (int r = 0; r < 2; ++r) {
      const int j = lane + 32 * r, a = jump[j];
      m[r] = out[j] | (a >= 0 ? out[a] : 0ull);
      jj[r] = a >= 0 ? jump[a] : -1;
    }
    __syncwarp();
    for (int r = 0; r < 2; ++r) {
      out[lane + 32 * r] = m[r];
      jump[lane + 32 * r] = jj[r];
    }
    __syncwarp();
  }
}

// One CTA per (q-head, node, sequence); a warp walks every kWarps-th row with an
// online softmax, the warps are merged at the end.
template <typename T>
__global__ void __launch_bounds__(kWarps * 32) tree_simple_kernel(const __grid_constant__ TreeParams p) {
  __shared__ uint64_t masks[64];
  __shared__ int jump[64];
  __shared__ float wm[kWarps], wl[kWarps], wacc[kWarps][256];
  pdl_launch_dependents();
  pdl_wait();
  const int h = blockIdx.x, node = blockIdx.y, b = blockIdx.z, lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int count = min(max(p.counts ? p.counts[b] : p.n, 0), p.n);
  if (node >= count) return;
  const int len = max(0, min(p.lens[b], p.n_ctx - count));
  if (w == 0) tree_masks(p.parents + (int64_t)b * p.n, count, masks, jump);
  __syncthreads();
  const uint64_t mask = masks[node];
  const T* q = static_cast<const T*>(p.q) + b * p.q_batch + node * p.q_node + h * p.q_head;
  const T* k = static_cast<const T*>(p.k) + b * p.kv_batch + (h / (p.H / p.HK)) * p.kv_head;
  const T* v = static_cast<const T*>(p.v) + b * p.kv_batch + (h / (p.H / p.HK)) * p.kv_head;
  float qr[8], acc[8], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    qr[r] = lane + 32 * r < p.D ? to_f32(q[lane + 32 * r]) : 0.f;
    acc[r] = 0.f;
  }
  for (int row = w; row < len + count; row += kWarps) {
    if (row >= len && !((mask >> (row - len)) & 1)) continue;
    const T* kr = k + row * p.kv_row;
    const T* vr = v + row * p.kv_row;
    float d = 0.f;
#pragma unroll
    for (int r = 0; r < 8; ++r)
      if (lane + 32 * r < p.D) d = fmaf(qr[r], to_f32(kr[lane + 32 * r]), d);
    const float s = warp_sum(d) * p.scale, mn = fmaxf(m, s), cf = m == -INFINITY ? 0.f : expf(m - mn), pf = expf(s - mn);
    l = l * cf + pf;
#pragma unroll
    for (int r = 0; r < 8; ++r)
      if (lane + 32 * r < p.D) acc[r] = fmaf(pf, to_f32(vr[lane + 32 * r]), acc[r] * cf);
    m = mn;
  }
  if (lane == 0) wm[w] = m, wl[w] = l;
#pragma unroll
  for (int r = 0; r < 8; ++r)
    if (lane + 32 * r < p.D) wacc[w][lane + 32 * r] = acc[r];
  __syncthreads();
  float M = -INFINITY, L = 0.f;
  for (int i = 0; i < kWarps; ++i) M = fmaxf(M, wm[i]);
  for (int i = 0; i < kWarps; ++i) L += wl[i] != 0.f ? wl[i] * expf(wm[i] - M) : 0.f;
  T* o = static_cast<T*>(p.o) + b * p.o_batch + node * p.o_node + h * p.o_head;
  for (int i = threadIdx.x; i < p.D; i += kWarps * 32) {
    float a = 0.f;
    for (int j = 0; j < kWarps; ++j) a += wl[j] != 0.f ? wacc[j][i] * expf(wm[j] - M) : 0.f;
    o[i] = from_f32<T>(a / L);
  }
}

bool tree_sizes_ok(int B, int n, int H, int HK, int D, int n_ctx) {
  return B >= 0 && B <= 65535 && n >= 1 && n <= BTF_TREE_MAX_NODES && HK >= 1 && H >= HK && H % HK == 0 &&
         H <= 65535 && D >= 8 && D <= 256 && D % 8 == 0 && n_ctx >= n;
}

}  // namespace
}  // namespace btf

using namespace btf;

extern "C" {

int64_t btf_tree_attention_work(int B, int n, int H, int HK, int D, int n_ctx) {
  if (!tree_sizes_ok(B, n, H, HK, D, n_ctx)) {
    fail(BTF_ERR_ARG, "btf_tree_attention_work: bad sizes");
    return -1;
  }
  return 256;
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
  if (!std::isfinite(a->scale)) return fail(BTF_ERR_ARG, "btf_tree_attention: scale must be finite");
  if (a->work_bytes < btf_tree_attention_work(a->B, a->n, a->H, a->HK, a->D, a->n_ctx) || !a->work ||
      reinterpret_cast<uintptr_t>(a->work) % 256)
    return fail(BTF_ERR_ARG, "btf_tree_attention: workspace too small, null or not 256-byte aligned");
  const DeviceInfo* dev = current_device();
  if (!dev) return BTF_ERR_STATE;
  const TreeParams p{a->q, a->k, a->v, a->o, a->q_batch, a->q_node, a->q_head, a->kv_batch, a->kv_row, a->kv_head,
                     a->o_batch, a->o_node, a->o_head, a->n, a->H, a->HK, a->D, a->n_ctx, a->lens, a->parents,
                     a->counts, a->scale};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 grid(a->H, a->n, a->B);
  const cudaError_t e = a->type == BTF_F16
                            ? launch_pdl(tree_simple_kernel<__half>, grid, dim3(kWarps * 32), 0, st, p)
                            : launch_pdl(tree_simple_kernel<__nv_bfloat16>, grid, dim3(kWarps * 32), 0, st, p);
  return e == cudaSuccess ? BTF_OK : cuda_fail(e, "btf_tree_attention");
}

}  // extern "C"
