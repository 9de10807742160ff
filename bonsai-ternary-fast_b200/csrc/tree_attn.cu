// Attention for a tree of drafted tokens over a cache (btf_tree_attention): which
// rows each CTA takes of the kernel of attn.cuh, and where the join finds their parts.
#include <algorithm>
#include <cmath>

#include "attn.cuh"

namespace btf {
namespace {

// One sequence's tiles after another's: CTA x has M tile x % mtiles of range x / mtiles. The parts:
// [mtiles][2 ranges][128].
struct TreeSegments : Segments {
  using Params = AttnParams;
  using Place = RowPlace;
  static constexpr int kMaps = 2;
  __device__ __forceinline__ TreeSegments(const AttnParams& p, bool warp0)
      : Segments(p, blockIdx.x, p.ranges, 0, blockIdx.x == 0 && warp0) {}
  __device__ __forceinline__ bool whole() const { return nt == seq.tiles; }
  __device__ __forceinline__ bool tree() const { return true; }
  __device__ __forceinline__ int map() const { return 0; }
  __device__ __forceinline__ int64_t slot() const { return ((int64_t)mt * 2 * ranges + 2 * range + (tile == 0)) * kRowsM; }
  __device__ __forceinline__ RowPlace place(int r, bool) const { return place_of(r); }

  // Where the parts of an output row lie.
  struct Parts {
    int n;
    int64_t base;
    __device__ __forceinline__ Parts(const AttnParams& p, const Seq& seq, int b, int node, int head) {
      const int G = p.H / p.HK, rr = node * G + head % G;
      const int r0 = ranges_of(p, 0, seq, b, head / G, &n);
      base = ((int64_t)(rr / kRowsM) * 2 * p.ranges + 2 * r0) * kRowsM + rr % kRowsM;
      if (n == 1) n = 0;  // written whole
    }
    __device__ __forceinline__ int64_t operator()(int s) const { return base + (2 * s + (s == 0)) * kRowsM; }
  };
};

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

template <typename T, int DP>
cudaError_t launch_tree(const AttnMaps<2>& maps, const AttnParams& p, cudaStream_t st) {
  return launch_pdl(attn_kernel<T, DP, TreeSegments>, dim3((unsigned)(p.ranges * p.mtiles)), dim3(kThreads),
                    (size_t)Cfg<DP>::kSmem, st, maps, p);
}
template <typename T>
cudaError_t launch_tree_d(const AttnMaps<2>& maps, const AttnParams& p, int sms, cudaStream_t st) {
  const cudaError_t e = p.D <= 64    ? launch_tree<T, 64>(maps, p, st)
                        : p.D <= 128 ? launch_tree<T, 128>(maps, p, st)
                        : p.D <= 192 ? launch_tree<T, 192>(maps, p, st)
                                     : launch_tree<T, 256>(maps, p, st);
  if (e != cudaSuccess || p.ranges == 1) return e;
  const int64_t rows = (int64_t)p.B * p.n * p.H;  // at most INT32_MAX
  // a CTA per row while all of them are resident at once
  if (rows <= 8 * sms) return launch_pdl(attn_join_kernel<T, 8, TreeSegments>, dim3((unsigned)rows), dim3(kJoinThreads), 0, st, p);
  return launch_pdl(attn_join_kernel<T, 1, TreeSegments>, dim3((unsigned)((rows + 7) / 8)), dim3(kJoinThreads), 0, st, p);
}

// The join runs between two launches that take all of shared memory: it asks for
// the same split of the SM's storage, which changes only on an idle SM.
template <typename T, int WARPS>
cudaError_t join_carveout() {
  return cudaFuncSetAttribute(attn_join_kernel<T, WARPS, TreeSegments>, cudaFuncAttributePreferredSharedMemoryCarveout,
                              cudaSharedmemCarveoutMaxShared);
}
template <typename T, int DP>
cudaError_t allow_smem(const DeviceInfo& d) {
  static_assert(Cfg<DP>::kSmem * Cfg<DP>::kPerSm <= 228 * 1024 - 1024 * Cfg<DP>::kPerSm);
  if (Cfg<DP>::kSmem > d.optin_smem) return cudaErrorInvalidValue;
  return cudaFuncSetAttribute(attn_kernel<T, DP, TreeSegments>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<DP>::kSmem);
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
  if (int rc = attn_args_ok(a, "btf_tree_attention")) return rc;
  if (a->B == 0) return BTF_OK;
  const DeviceInfo* dev = current_device();
  if (!dev) return BTF_ERR_STATE;
  const Plan plan = tree_plan(*dev, a->B, a->n, a->H, a->HK, a->D, a->n_ctx);
  if (a->work_bytes < plan.bytes)
    return fail(BTF_ERR_ARG, "btf_tree_attention: the workspace has %lld bytes, %lld are needed", (long long)a->work_bytes,
                (long long)plan.bytes);
  if (plan.ranges > 1024 || attn_too_many(*a))
    return fail(BTF_ERR_UNSUPPORTED, "btf_tree_attention: too many sequences and heads for one launch");
  const bool b_one = a->B == 1 || a->kv_batch == 0, h_one = a->HK == 1 || a->kv_head == 0;
  AttnMaps<2> maps;
  if (int rc = encode_own(&maps.m[0], *a, "btf_tree_attention")) return rc;
  uint8_t* work = static_cast<uint8_t*>(a->work);
  const AttnParams p{a->q, a->v, a->o, a->q_batch, a->q_node, a->q_head, a->kv_batch, a->kv_row, a->kv_head, a->o_batch,
                     a->o_node, a->o_head, a->B, a->n, a->H, a->HK, a->D, a->n_ctx, plan.mtiles, plan.ranges,
                     b_one ? 0 : 1, h_one ? 0 : 1, a->lens, a->parents, a->counts,
                     std::max(std::fabs(a->scale) * 1.4426950408889634f, 0x1p-100f), a->scale < 0 ? 0x80008000u : 0u,
                     reinterpret_cast<int32_t*>(work), reinterpret_cast<float*>(work + plan.off_part),
                     reinterpret_cast<float*>(work + plan.off_ml), dev->err_word};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e =
      a->type == BTF_F16 ? launch_tree_d<__half>(maps, p, dev->sm_count, st)
                              : launch_tree_d<__nv_bfloat16>(maps, p, dev->sm_count, st);
  return e == cudaSuccess ? BTF_OK : cuda_fail(e, "btf_tree_attention");
}

}  // extern "C"
