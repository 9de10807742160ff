// Attention for a batch whose sequences share their first rows (btf_prefix_attention):
// a system prompt, a document, the prompt of several answers.
//
//   o = (sum_j p_j v_j over the shared rows + the own rows) / (sum_j p_j over both)
//
// The shared rows are read once for all sequences: their q rows, of every live node and
// of the G q-heads of a kv-head, are the rows of one matrix, 128 to an M tile, and a part
// of the softmax (maximum, sum, O) comes out for each. The own rows and the tree are
// btf_tree_attention's work and kernel (attn.cuh), and leave parts likewise; a second
// kernel joins them. Nodes that a sequence does not have take no rows of an M tile.
//
// Work: a share of the CTAs takes the shared rows, the others the own ones, by the tiles
// that either has and how they come out in whole segments (Split). A CTA of the shared
// rows takes one or several of equal stretches of (kv-head, M tile); neighbours have the
// same rows of K and V and different M tiles, so that those come from L2.
//
// What bounds it. Few rows: latency, as in attn.cuh. Many M tiles: a tile of 64 rows is bound by what the tensor cores read
// of shared memory, 96 KB at D = 128 with the tile's arrival (768 cycles, 512 of them the MMAs) and as in attn.cuh at D =
// 256 (1560); each segment's ways in and out come on top, one after another, since nothing of the next segment begins before
// the last one's O is out. Measured (device time; cycles of a CTA's softmax warps, on average, from the wait on):
//   4 sequences over 1000 shared rows, 24/4 fp16 heads of 256: 16.9 us.
//   48 over 4099, 20/5 bf16 heads of 96: 23.5 us. A CTA of the shared rows has 5 tiles, 7.4 of 21 thousand cycles (the
//     split 4, q's way in 5.4, the first S 1.1, the way out 2.6); one of own rows 1.5 segments of a tile, 4 of 20 (6.2, 3.6,
//     1.6, 2.6); the rest of the time is the launches and the join.
//   16 of 8 nodes over 16384 and up to 1100 own, 24/4 fp16 heads of 256: 59 to 64 us (29 GFLOP, 480 TFLOP/s). The shared rows'
//     26 tiles take 45 of 73 thousand cycles, 1750 each; q's way in 16, the split 4, the way out 5; the join comes behind.
//   128 over 65536 and up to 2000 own, 32/8 bf16 heads of 128: 171 to 203 us (138 GFLOP, 680 to 810 TFLOP/s; own rows read by
//     each sequence would be 34 GB). The shared rows' 146 tiles take 239 of 259 thousand cycles, 1630 each with two CTAs an
//     SM, at 1.4 to 1.6 GHz under the power cap; a quarter of the CTAs has own rows, 15 segments each, whose ways in and out
//     are 85 of 228 thousand cycles.
#include "attn.cuh"

namespace btf {
namespace {

constexpr int kMaxChunks = 32;   // stretches of the shared rows: what a warp compares, a lane each
constexpr int kSegTiles = 5;     // what a segment costs beside its tiles: q's way in and O's way out

struct PrefixParams : AttnParams {
  const int32_t* prefix_len;  // or null: all
  int prefix_rows, prefix_h;  // prefix_h: 0: every kv-head has the same shared rows
  int ctas, most_mtiles, most_chunks;
  int rpad;                    // rows of a part of own rows
  int64_t own_part, own_whole; // first rows of the parts of cut, and of whole, pairs
};

// How the CTAs are shared out; the same in every warp.
struct Split {
  int len, tiles, nodes;     // shared rows and their tiles; live nodes of the batch
  int mtiles, chunks, ctas;  // M tiles of the shared rows, stretches of each, CTAs for them
  int ranges;                // of the own rows
  __device__ __forceinline__ explicit Split(const PrefixParams& p) {
    const int lane = threadIdx.x & 31;
    len = p.prefix_len ? min(max(*p.prefix_len, 0), p.prefix_rows) : p.prefix_rows;
    int own = 0, pairs = 0;  // tiles of the own rows of a kv-head, sequences with any
    nodes = 0;
    for (int b0 = 0; b0 < p.B; b0 += 32) {
      Seq s;
      s.count = s.tiles = 0;
      if (b0 + lane < p.B) s = Seq(p, b0 + lane);
      nodes += __reduce_add_sync(0xffffffffu, s.count);
      own += __reduce_add_sync(0xffffffffu, s.tiles);
      pairs += __popc(__ballot_sync(0xffffffffu, s.tiles > 0));
    }
    tiles = (len + kTile - 1) / kTile;
    mtiles = (int)(((int64_t)nodes * (p.H / p.HK) + kRowsM - 1) / kRowsM);
    chunks = ctas = 0;
    ranges = p.ctas / p.mtiles;
    if (tiles == 0 || mtiles == 0) return;
    // lane i: the shared rows of each (kv-head, M tile) in i + 1 stretches
    const float streams = (float)p.HK * (float)mtiles;
    const float mine = (float)p.HK * (float)p.mtiles * ((float)own + (float)(kSegTiles * pairs));
    // and what the slowest CTA then has, with the CTAs shared out so that both kinds end together: in w turns over
    // the shared rows' items, rounded down or up
    const int n = min(lane + 1, min(p.most_chunks, tiles));
    const float items = streams * (float)n, each = ceilf((float)tiles / (float)n) + kSegTiles;
    const float most = (float)(p.ctas - p.mtiles), w = floorf((mine + items * each) / (each * (float)p.ctas));
    float take = 0.f, cost = INFINITY;
#pragma unroll
    for (int up = 0; up < 2; ++up) {
      const float t = fminf(most, ceilf(items / fmaxf(1.0f, w + (float)up)));
      const float c = fmaxf(ceilf(items / t) * each, mine / ((float)p.ctas - t));
      if (c < cost) cost = c, take = t;
    }
    const uint32_t best = __reduce_min_sync(0xffffffffu, __float_as_uint(cost));
    const int l = __ffs(__ballot_sync(0xffffffffu, __float_as_uint(cost) == best)) - 1;
    chunks = __shfl_sync(0xffffffffu, n, l);
    ctas = __shfl_sync(0xffffffffu, (int)take, l);
    ranges = (p.ctas - ctas) / p.mtiles;
  }
};

// CTAs below Split::ctas take stretches of the shared rows, the others Segments of the own ones. The table for the
// join, behind that of Segments: stretches, the own rows' ranges, then each sequence's first live node.
struct PrefixSegments : Segments {
  using Params = PrefixParams;
  using Place = RowPlace;
  static constexpr int kMaps = 4;
  const PrefixParams& pp;
  const Split sp;
  const bool shared;  // whether this CTA's segments are of the shared rows
  int item, chunk, pmt;

  __device__ __forceinline__ PrefixSegments(const PrefixParams& p_, bool warp0) : PrefixSegments(p_, warp0, Split(p_)) {}
  __device__ __forceinline__ PrefixSegments(const PrefixParams& p_, bool warp0, const Split& s)
      : Segments(p_, (int)blockIdx.x < s.ctas || (int)blockIdx.x >= s.ctas + s.ranges * p_.mtiles ? -1 : (int)blockIdx.x - s.ctas,
                 s.ranges, kSegTiles, warp0 && (int)blockIdx.x == s.ctas),
        pp(p_), sp(s), shared((int)blockIdx.x < s.ctas), item((int)blockIdx.x), chunk(0), pmt(0) {
    if (shared) take();
    if (warp0 && (int)blockIdx.x == sp.ctas) {
      const int lane = threadIdx.x & 31;
      if (lane == 0) p.first[p.B + 2] = sp.chunks, p.first[p.B + 3] = sp.ranges;
      int before = 0;
      for (int b0 = 0; b0 < p.B; b0 += 32) {
        const int t = running(b0);
        if (b0 + lane < p.B) p.first[p.B + 4 + b0 + lane] = before + t - count_of(b0 + lane);
        before += __shfl_sync(0xffffffffu, t, 31);
      }
    }
  }
  __device__ __forceinline__ int count_of(int i) const { return i >= p.B ? 0 : p.counts ? min(max(p.counts[i], 0), p.n) : p.n; }
  // Live nodes of the sequences from b0 up to this lane's.
  __device__ __forceinline__ int running(int b0) const {
    const int lane = threadIdx.x & 31;
    int t = count_of(b0 + lane);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int q = __shfl_up_sync(0xffffffffu, t, o);
      if (lane >= o) t += q;
    }
    return t;
  }
  __device__ __forceinline__ void take() {
    nt = 0;
    if ((int64_t)item >= (int64_t)p.HK * sp.chunks * sp.mtiles) return;
    pmt = item % sp.mtiles;
    chunk = item / sp.mtiles % sp.chunks;
    kvh = item / sp.mtiles / sp.chunks;
    tile = (int)((int64_t)chunk * sp.tiles / sp.chunks);
    nt = (int)((int64_t)(chunk + 1) * sp.tiles / sp.chunks) - tile;
    seq.count = 0, seq.len = sp.len, seq.tiles = sp.tiles;
  }
  __device__ __forceinline__ void next() {
    if (!shared) return Segments::next();
    item += sp.ctas;
    take();
  }
  __device__ __forceinline__ int rows() const {
    return shared ? (int)min((int64_t)kRowsM, (int64_t)sp.nodes * (p.H / p.HK) - (int64_t)pmt * kRowsM) : Segments::rows();
  }
  __device__ __forceinline__ bool whole() const { return sp.tiles == 0 && nt == seq.tiles; }
  __device__ __forceinline__ bool tree() const { return !shared; }
  __device__ __forceinline__ int map() const { return shared ? 2 : 0; }
  __device__ __forceinline__ int plane_b() const { return shared ? 0 : Segments::plane_b(); }
  __device__ __forceinline__ int plane_h() const { return shared ? kvh * pp.prefix_h : Segments::plane_h(); }
  static __device__ __forceinline__ int64_t shared_slot(const PrefixParams& p, int chunk, int kvh, int mt) {
    return (((int64_t)chunk * p.HK + kvh) * p.most_mtiles + mt) * kRowsM;
  }
  __device__ __forceinline__ int64_t slot() const {
    if (shared) return shared_slot(pp, chunk, kvh, pmt);
    if (nt == seq.tiles) return pp.own_whole + (((int64_t)b * p.HK + kvh) * p.mtiles + mt) * pp.rpad;
    return pp.own_part + ((int64_t)mt * 2 * ranges + 2 * range + (tile == 0)) * pp.rpad;
  }
  __device__ __forceinline__ RowPlace place(int r, bool on) const {
    if (!shared) return place_of(r);
    const int G = p.H / p.HK;
    const bool live = r < rows();
    const int64_t rr = (int64_t)pmt * kRowsM + (live ? r : 0);
    int node = (int)(rr / G), seq_b = 0;
    const int head = kvh * G + (int)(rr % G);
    if (!p.counts) {
      seq_b = node / p.n;
      node %= p.n;
    } else if (on) {  // (of the whole warp) the sequence in whose live nodes this one is
      bool found = false;
      for (int b0 = 0; b0 < p.B; b0 += 32) {
        const int t = running(b0), all = __shfl_sync(0xffffffffu, t, 31);
        int at = 0;  // lanes whose running number is not above the node
#pragma unroll
        for (int step = 16; step; step >>= 1) {
          const int v = __shfl_sync(0xffffffffu, t, at + step - 1);
          if (v <= node) at += step;
        }
        const int before = __shfl_sync(0xffffffffu, t, at > 0 ? at - 1 : 0);
        if (!found && node < all) {
          found = true;
          seq_b = b0 + at;
          node -= at > 0 ? before : 0;
        } else if (!found) {
          node -= all;
        }
        if (__all_sync(0xffffffffu, found)) break;
      }
    }
    return {seq_b, node, head, live && seq_b < p.B};
  }

  struct Parts {
    int n, shared, own;
    int64_t own_base, own_step, shared_base, shared_step;
    __device__ __forceinline__ Parts(const PrefixParams& p, const Seq& seq, int b, int node, int head) {
      const int G = p.H / p.HK, kvh = head / G, rr = node * G + head % G, mt = rr / kRowsM;
      shared = p.first[p.B + 2];
      const int ranges = p.first[p.B + 3];
      const int64_t ps = ((int64_t)p.first[p.B + 4 + b] + node) * G + head % G;
      shared_base = shared_slot(p, 0, kvh, (int)(ps / kRowsM)) + ps % kRowsM;
      shared_step = shared_slot(p, 1, 0, 0);
      const int r0 = ranges_of(p, kSegTiles, seq, b, kvh, &own);
      own_step = 2 * p.rpad;
      own_base = own == 1 ? p.own_whole + (((int64_t)b * p.HK + kvh) * p.mtiles + mt) * p.rpad + rr % kRowsM
                          : p.own_part + ((int64_t)mt * 2 * ranges + 2 * r0) * p.rpad + rr % kRowsM;
      n = shared == 0 && own == 1 ? 0 : shared + own;
    }
    __device__ __forceinline__ int64_t operator()(int s) const {
      if (s < shared) return shared_base + s * shared_step;
      s -= shared;
      return own_base + s * own_step + (own > 1 && s == 0 ? own_step / 2 : 0);
    }
  };
};

bool prefix_sizes_ok(int prefix_rows) { return prefix_rows >= 0 && prefix_rows <= (1 << 30); }

struct Plan {
  int mtiles, ctas, most_mtiles, most_chunks, rpad;
  int64_t own_part, own_whole, off_part, off_ml, bytes;
};
Plan prefix_plan(const DeviceInfo& d, int B, int n, int H, int HK, int D, int prefix_rows) {
  Plan r;
  const int G = H / HK;
  r.mtiles = (n * G + kRowsM - 1) / kRowsM;
  r.ctas = std::max(d.sm_count * (D <= 128 ? 2 : 1), r.mtiles + 1);
  r.most_mtiles = (int)(((int64_t)B * n * G + kRowsM - 1) / kRowsM);
  const int64_t tiles = ((int64_t)prefix_rows + kTile - 1) / kTile, streams = std::max<int64_t>(1, (int64_t)HK * r.most_mtiles);
  r.most_chunks = (int)std::max<int64_t>(1, std::min<int64_t>({kMaxChunks, tiles, (2 * r.ctas + streams - 1) / streams}));
  r.rpad = std::min(kRowsM, n * G);
  r.own_part = (int64_t)r.most_chunks * HK * r.most_mtiles * kRowsM;
  r.own_whole = r.own_part + (int64_t)r.mtiles * 2 * (r.ctas / r.mtiles) * r.rpad;
  const int64_t rows = r.own_whole + (int64_t)B * HK * r.mtiles * r.rpad;
  r.off_part = ((int64_t)(2 * B + 4) * 4 + 255) / 256 * 256;
  r.off_ml = r.off_part + rows * D * 4;
  r.bytes = r.off_ml + rows * 8;
  return r;
}

template <typename T, int DP>
cudaError_t launch_prefix(const AttnMaps<4>& maps, const PrefixParams& p, cudaStream_t st) {
  return launch_pdl(attn_kernel<T, DP, PrefixSegments>, dim3((unsigned)p.ctas), dim3(kThreads), (size_t)Cfg<DP>::kSmem, st,
                    maps, p);
}
template <typename T>
cudaError_t launch_prefix_d(const AttnMaps<4>& maps, const PrefixParams& p, int sms, cudaStream_t st) {
  const cudaError_t e = p.D <= 64    ? launch_prefix<T, 64>(maps, p, st)
                        : p.D <= 128 ? launch_prefix<T, 128>(maps, p, st)
                        : p.D <= 192 ? launch_prefix<T, 192>(maps, p, st)
                                     : launch_prefix<T, 256>(maps, p, st);
  if (e != cudaSuccess) return e;
  const int64_t rows = (int64_t)p.B * p.n * p.H;  // at most INT32_MAX
  if (rows <= 4 * sms)  // a CTA a row while they are few (960 rows of 96: 26.8 us so, 23.4 with a warp a row)
    return launch_pdl(attn_join_kernel<T, 8, PrefixSegments>, dim3((unsigned)rows), dim3(kJoinThreads), 0, st, p);
  return launch_pdl(attn_join_kernel<T, 1, PrefixSegments>, dim3((unsigned)((rows + 7) / 8)), dim3(kJoinThreads), 0, st, p);
}

// (the join: the same split of the SM's storage as the launches around it, which changes only on an idle SM)
template <typename T, int WARPS>
cudaError_t join_carveout() {
  return cudaFuncSetAttribute(attn_join_kernel<T, WARPS, PrefixSegments>, cudaFuncAttributePreferredSharedMemoryCarveout,
                              cudaSharedmemCarveoutMaxShared);
}
template <typename T, int DP>
cudaError_t allow_smem(const DeviceInfo& d) {
  if (Cfg<DP>::kSmem > d.optin_smem) return cudaErrorInvalidValue;
  return cudaFuncSetAttribute(attn_kernel<T, DP, PrefixSegments>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<DP>::kSmem);
}

}  // namespace

int prefix_attn_setup(DeviceInfo& d) {
  for (cudaError_t e : {allow_smem<__half, 64>(d), allow_smem<__half, 128>(d), allow_smem<__half, 192>(d),
                        allow_smem<__half, 256>(d), allow_smem<__nv_bfloat16, 64>(d), allow_smem<__nv_bfloat16, 128>(d),
                        allow_smem<__nv_bfloat16, 192>(d), allow_smem<__nv_bfloat16, 256>(d),
                        join_carveout<__half, 1>(), join_carveout<__half, 8>(), join_carveout<__nv_bfloat16, 1>(),
                        join_carveout<__nv_bfloat16, 8>()})
    if (e != cudaSuccess) return cuda_fail(e, "the attention kernels' attributes");
  return BTF_OK;
}

}  // namespace btf

using namespace btf;

extern "C" {

int64_t btf_prefix_attention_work(int B, int n, int H, int HK, int D, int n_ctx, int prefix_rows) {
  if (!tree_sizes_ok(B, n, H, HK, D, n_ctx) || !prefix_sizes_ok(prefix_rows)) {
    fail(BTF_ERR_ARG, "btf_prefix_attention_work: bad sizes (B %d, n %d, H %d, HK %d, D %d, n_ctx %d, %d shared rows)", B, n, H,
         HK, D, n_ctx, prefix_rows);
    return -1;
  }
  const DeviceInfo* dev = current_device();
  if (!dev) return -1;
  return prefix_plan(*dev, B, n, H, HK, D, prefix_rows).bytes;
}

int btf_prefix_attention(const btf_tree_attn* a, const btf_prefix* s, void* stream) {
  const char* what = "btf_prefix_attention";
  if (!s) return fail(BTF_ERR_ARG, "%s: null arguments", what);
  if (int rc = attn_args_ok(a, what)) return rc;
  if (!prefix_sizes_ok(s->rows)) return fail(BTF_ERR_ARG, "%s: need 0..2^30 shared rows (got %d)", what, s->rows);
  if (a->B == 0) return BTF_OK;
  auto al = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  if (s->rows > 0) {
    if (!s->k || !s->v || !al(s->k) || !al(s->v))
      return fail(BTF_ERR_ARG, "%s: the shared k or v is null or not 16-byte aligned", what);
    if (s->row < 0 || s->row % 8 || s->head < 0 || s->head % 8)
      return fail(BTF_ERR_ARG, "%s: strides must be multiples of 8 elements, >= 0", what);
    if (s->rows > 1 && s->row == 0) return fail(BTF_ERR_ARG, "%s: the shared rows need a stride", what);
  }
  const DeviceInfo* dev = current_device();
  if (!dev) return BTF_ERR_STATE;
  const Plan plan = prefix_plan(*dev, a->B, a->n, a->H, a->HK, a->D, s->rows);
  if (a->work_bytes < plan.bytes)
    return fail(BTF_ERR_ARG, "%s: the workspace has %lld bytes, %lld are needed", what, (long long)a->work_bytes,
                (long long)plan.bytes);
  if (plan.ctas > 1024 || attn_too_many(*a) || (int64_t)a->HK * plan.most_mtiles * plan.most_chunks > INT32_MAX / 2 ||
      (int64_t)a->B * a->HK * ((a->n_ctx + kTile - 1) / kTile + kSegTiles) > INT32_MAX / 2)
    return fail(BTF_ERR_UNSUPPORTED, "%s: too many sequences and heads for one launch", what);
  const int heads = s->head == 0 ? 1 : a->HK;
  AttnMaps<4> maps;
  if (int rc = encode_own(&maps.m[0], *a, what)) return rc;
  if (s->rows > 0) {
    if (int rc = encode_rows(&maps.m[2], a->type, s->k, a->D, s->rows, heads, 1, s->row, s->head, 0, what)) return rc;
    if (int rc = encode_rows(&maps.m[3], a->type, s->v, a->D, s->rows, heads, 1, s->row, s->head, 0, what)) return rc;
  } else {
    maps.m[2] = maps.m[0], maps.m[3] = maps.m[1];
  }
  uint8_t* work = static_cast<uint8_t*>(a->work);
  PrefixParams p{};
  static_cast<AttnParams&>(p) = {
      a->q, a->v, a->o, a->q_batch, a->q_node, a->q_head, a->kv_batch, a->kv_row, a->kv_head, a->o_batch,
      a->o_node, a->o_head, a->B, a->n, a->H, a->HK, a->D, a->n_ctx, plan.mtiles, 0,
      a->B == 1 || a->kv_batch == 0 ? 0 : 1, a->HK == 1 || a->kv_head == 0 ? 0 : 1, a->lens, a->parents, a->counts,
      std::max(std::fabs(a->scale) * 1.4426950408889634f, 0x1p-100f), a->scale < 0 ? 0x80008000u : 0u,
      reinterpret_cast<int32_t*>(work), reinterpret_cast<float*>(work + plan.off_part),
      reinterpret_cast<float*>(work + plan.off_ml), dev->err_word};
  p.prefix_len = s->len, p.prefix_rows = s->rows, p.prefix_h = heads > 1;
  p.ctas = plan.ctas, p.most_mtiles = plan.most_mtiles, p.most_chunks = plan.most_chunks, p.rpad = plan.rpad;
  p.own_part = plan.own_part, p.own_whole = plan.own_whole;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = a->type == BTF_F16 ? launch_prefix_d<__half>(maps, p, dev->sm_count, st)
                                           : launch_prefix_d<__nv_bfloat16>(maps, p, dev->sm_count, st);
  return e == cudaSuccess ? BTF_OK : cuda_fail(e, what);
}

}  // extern "C"
