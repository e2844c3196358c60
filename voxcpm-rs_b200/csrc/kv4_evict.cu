// Eviction from the 4-bit KV cache by accumulated attention weight (vx_kv4_evict).
//
// One cluster of C thread blocks per (sequence, KV head).  A row's rank is its weight as an
// ordered 32-bit key (protected rows: the largest key); four 8-bit radix passes over the keys
// find the key T of the keep-th largest row and how many rows of key T stay (those of the lowest
// slots).  Attention does not depend on the order of rows, so nothing is shifted: the i-th slot
// below `keep` that became free takes the i-th kept row behind it.  Sources (slots >= keep) and
// destinations (slots < keep) are disjoint, so the moves need no order among them.
#include <cooperative_groups.h>

#include "common.cuh"
#include "kv4.cuh"
#include "runtime.cuh"

namespace cg = cooperative_groups;

namespace vx {
namespace {

constexpr int EV_THREADS = 1024;
constexpr int EV_MAX_CLUSTER = 8;
constexpr int EV_MAX_LEN = 131072;

struct EvictArgs {
  uint8_t *k_codes, *k_scales, *v_codes, *v_scales;
  const float* weights;
  const int64_t* positions;
  float* weights_out;
  int64_t* positions_out;
  const int *lens, *seen;
  int* lens_out;
  int B, nkv, d, cap, max_len, keep, sink, recent, seg_max;
  int* err;
};

// Rank of a row: larger weight, larger key; -0 counts as 0 and a NaN as the largest weight.
__device__ __forceinline__ uint32_t weight_key(float w) {
  const uint32_t u = __float_as_uint(w + 0.f);
  if (w != w) return 0xfffffffeu;
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__global__ void __launch_bounds__(EV_THREADS) kv4_evict_kernel(const EvictArgs a) {
  extern __shared__ __align__(16) uint32_t dyn[];  // keys [seg_max], then slot lists
  __shared__ uint32_t hist[2][256], tot[256];
  __shared__ uint32_t warp_n[32], sh[8];
  cg::cluster_group cl = cg::this_cluster();
  const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  const int unit = blockIdx.x / C, b = unit / a.nkv, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int n = a.lens[b];
  const size_t row0 = (size_t)unit * a.cap;
  if (n < 0 || n > a.max_len) {  // the same for every block of the cluster
    if (unit % a.nkv == 0 && rank == 0 && tid == 0) {
      record_error(a.err, VX_DEVICE_ERR_BOUNDS);
      a.lens_out[b] = n;
    }
    return;
  }
  if (unit % a.nkv == 0 && rank == 0 && tid == 0) a.lens_out[b] = min(n, a.keep);
  if (a.keep == 0) return;  // every row goes
  if (n <= a.keep) {  // nothing to let go of
    for (int j = rank * EV_THREADS + tid; j < n; j += C * EV_THREADS) {
      if (a.weights_out != a.weights) a.weights_out[row0 + j] = a.weights[row0 + j];
      if (a.positions_out != a.positions) a.positions_out[row0 + j] = a.positions[row0 + j];
    }
    return;
  }
  const int seg = (n + C - 1) / C, lo = min(n, rank * seg), hi = min(n, lo + seg), cnt = hi - lo;
  uint32_t* keys = dyn;
  uint32_t* list = dyn + a.seg_max;  // this block's free slots from the front, its movers from the back
  const int64_t since = (int64_t)a.seen[b] - a.recent;
  for (int j = tid; j < cnt; j += EV_THREADS) {
    const int64_t pos = a.positions[row0 + lo + j];
    keys[j] = (pos < a.sink || pos >= since) ? 0xffffffffu : weight_key(a.weights[row0 + lo + j]);
  }
  uint32_t prefix = 0, left = (uint32_t)a.keep;  // rows still to be found among the keys of this prefix
  for (int pass = 0; pass < 4; ++pass) {
    const int shift = 24 - 8 * pass;
    uint32_t* h = hist[pass & 1];
    if (tid < 256) h[tid] = 0;
    __syncthreads();
    for (int j = tid; j < cnt; j += EV_THREADS) {
      const uint32_t k = keys[j];
      if (pass == 0 || (k >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&h[(k >> shift) & 255], 1u);
    }
    cl.sync();
    if (tid < 256) {
      uint32_t t = 0;
      for (int r = 0; r < C; ++r) t += cl.map_shared_rank(h, r)[tid];
      tot[tid] = t;
    }
    __syncthreads();
    if (warp == 0) {  // the digit at which the count from above reaches `left`
      uint32_t v[8], s = 0;
      for (int e = 0; e < 8; ++e) s += v[e] = tot[255 - (lane * 8 + e)];
      uint32_t incl = s;
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t t = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += t;
      }
      uint32_t above = incl - s;
      if (above < left && incl >= left) {
        int e = 0;
        while (above + v[e] < left) above += v[e++];
        sh[0] = prefix | ((uint32_t)(255 - (lane * 8 + e)) << shift);
        sh[1] = left - above;
      }
    }
    __syncthreads();
    prefix = sh[0];
    left = sh[1];
  }
  const uint32_t T = prefix, ties = left;  // `ties` rows of key T stay, in slot order

  // how many rows of key T lie in the blocks before this one
  uint32_t c = 0;
  for (int j = tid; j < cnt; j += EV_THREADS) c += keys[j] == T;
  c = __reduce_add_sync(0xffffffffu, c);
  if (lane == 0) warp_n[warp] = c;
  __syncthreads();
  if (warp == 0) {
    c = __reduce_add_sync(0xffffffffu, warp_n[lane]);
    if (lane == 0) sh[2] = c;
  }
  cl.sync();
  uint32_t eq_base = 0;
  for (int r = 0; r < rank; ++r) eq_base += *cl.map_shared_rank(&sh[2], r);

  // free slots and movers of this block, in slot order
  uint32_t holes = 0, movers = 0;
  for (int j0 = 0; j0 < cnt; j0 += EV_THREADS) {
    const int j = j0 + tid, slot = lo + j;
    const bool in = j < cnt;
    const uint32_t k = in ? keys[j] : 0;
    const uint32_t eq = __ballot_sync(0xffffffffu, in && k == T);
    __syncthreads();
    if (lane == 0) warp_n[warp] = __popc(eq);
    __syncthreads();
    uint32_t before = 0, all = 0;
    for (int w = 0; w < 32; ++w) {
      if (w < warp) before += warp_n[w];
      all += warp_n[w];
    }
    const uint32_t tr = eq_base + before + __popc(eq & ((1u << lane) - 1));
    eq_base += all;
    const bool stays = in && (k > T || (k == T && tr < ties));
    const bool hole = in && slot < a.keep && !stays, mover = stays && slot >= a.keep;
    const uint32_t hb = __ballot_sync(0xffffffffu, hole), mb = __ballot_sync(0xffffffffu, mover);
    __syncthreads();
    if (lane == 0) warp_n[warp] = __popc(hb) | (__popc(mb) << 16);
    __syncthreads();
    before = all = 0;
    for (int w = 0; w < 32; ++w) {
      if (w < warp) before += warp_n[w];
      all += warp_n[w];
    }
    const uint32_t below = (1u << lane) - 1;
    if (hole) list[holes + (before & 0xffff) + __popc(hb & below)] = slot;
    if (mover) list[a.seg_max - 1 - (movers + (before >> 16) + __popc(mb & below))] = slot;
    holes += all & 0xffff;
    movers += all >> 16;
    if (stays && slot < a.keep) {
      if (a.weights_out != a.weights) a.weights_out[row0 + slot] = a.weights[row0 + slot];
      if (a.positions_out != a.positions) a.positions_out[row0 + slot] = a.positions[row0 + slot];
    }
  }
  if (tid == 0) {
    sh[3] = holes;
    sh[4] = movers;
  }
  cl.sync();
  uint32_t m0 = 0, hole0[EV_MAX_CLUSTER + 1];
  hole0[0] = 0;
#pragma unroll
  for (int r = 0; r < EV_MAX_CLUSTER; ++r) {
    hole0[r + 1] = hole0[r];
    if (r < C) {
      if (r < rank) m0 += *cl.map_shared_rank(&sh[4], r);
      hole0[r + 1] += *cl.map_shared_rank(&sh[3], r);
    }
  }
  // 16 lanes move a row
  const int cb = a.d / 32, sb = a.d / 16;  // 16-byte pieces of the codes, bytes of the scales
  const int l16 = tid & 15;
  for (uint32_t i = tid >> 4; i < movers; i += EV_THREADS / 16) {
    const size_t src = row0 + list[a.seg_max - 1 - i];
    const uint32_t g = m0 + i;
    int owner = 0;
    uint32_t first = 0;
#pragma unroll
    for (int r = 1; r < EV_MAX_CLUSTER; ++r)
      if (g >= hole0[r]) {
        owner = r;
        first = hole0[r];
      }
    const size_t dst = row0 + cl.map_shared_rank(list, owner)[g - first];
    if (l16 < cb)
      reinterpret_cast<uint4*>(a.k_codes + dst * (a.d / 2))[l16] =
          reinterpret_cast<const uint4*>(a.k_codes + src * (a.d / 2))[l16];
    else if (l16 < 2 * cb)
      reinterpret_cast<uint4*>(a.v_codes + dst * (a.d / 2))[l16 - cb] =
          reinterpret_cast<const uint4*>(a.v_codes + src * (a.d / 2))[l16 - cb];
    else if (l16 < 2 * cb + sb / 4)
      reinterpret_cast<uint32_t*>(a.k_scales + dst * sb)[l16 - 2 * cb] =
          reinterpret_cast<const uint32_t*>(a.k_scales + src * sb)[l16 - 2 * cb];
    else if (l16 < 2 * cb + sb / 2)
      reinterpret_cast<uint32_t*>(a.v_scales + dst * sb)[l16 - 2 * cb - sb / 4] =
          reinterpret_cast<const uint32_t*>(a.v_scales + src * sb)[l16 - 2 * cb - sb / 4];
    else if (l16 == 14)
      a.weights_out[dst] = a.weights[src];
    else if (l16 == 15)
      a.positions_out[dst] = a.positions[src];
  }
  cl.sync();  // the lists are read by the other blocks
}

int cluster_of(int max_len) {
  int c = 1;
  while (c < EV_MAX_CLUSTER && max_len > 4096 * c) c *= 2;
  return c;
}

}  // namespace

cudaError_t kv4_evict_configure() {
  return cudaFuncSetAttribute(kv4_evict_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              EV_MAX_LEN / EV_MAX_CLUSTER * 8);
}

}  // namespace vx

using namespace vx;

extern "C" int vx_kv4_evict(vx_ctx* ctx, const vx_kv4* c, const int32_t* lens, const int32_t* seen, int max_len,
                            int keep, int sink, int recent, float* weights_out, int64_t* positions_out,
                            int32_t* lens_out, vx_stream stream) {
  const int rc = kv4_check(ctx, c, "kv4_evict");
  if (rc) return rc;
  if (!lens || !seen || !lens_out || !weights_out || !positions_out)
    return fail(ctx, VX_ERR_ARG, "kv4_evict: lens, seen and the outputs are needed");
  if (!c->weights || !c->positions) return fail(ctx, VX_ERR_ARG, "kv4_evict: the cache keeps no weights and positions");
  if (lens_out == lens) return fail(ctx, VX_ERR_ARG, "kv4_evict: lens_out must not be lens");
  if (max_len < 0 || max_len > c->capacity)
    return fail(ctx, VX_ERR_SHAPE, "kv4_evict: max_len %d outside 0..%d", max_len, c->capacity);
  if (max_len > EV_MAX_LEN) return fail(ctx, VX_ERR_SHAPE, "kv4_evict: max_len %d > %d", max_len, EV_MAX_LEN);
  if (keep < 0 || sink < 0 || recent < 0 || (long long)sink + recent > keep)
    return fail(ctx, VX_ERR_SHAPE, "kv4_evict: sink %d + recent %d must fit in keep %d", sink, recent, keep);
  DeviceGuard guard(ctx->device);
  const int C = cluster_of(max_len);
  const int seg = std::max(1, (max_len + C - 1) / C);
  const size_t smem = (size_t)seg * 2 * 4;
  EvictArgs a = {c->k_codes, c->k_scales, c->v_codes, c->v_scales, c->weights, c->positions, weights_out,
                 positions_out, lens, seen, lens_out, c->batch, c->n_kv_heads, c->head_dim, c->capacity, max_len, keep,
                 sink, recent, seg, ctx->dev_err};
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(c->batch * c->n_kv_heads * C);
  cfg.blockDim = dim3(EV_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = pick_stream(ctx, stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  count_launch();
  VX_CUDA(ctx, cudaLaunchKernelEx(&cfg, kv4_evict_kernel, a));
  return VX_OK;
}
