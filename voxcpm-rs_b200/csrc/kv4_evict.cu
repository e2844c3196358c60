// Eviction from the 4-bit KV cache by accumulated attention weight (vx_kv4_evict).
//
// One cluster of C thread blocks per (sequence, KV head).  A row's rank is its weight as an
// ordered 32-bit key (protected rows: the largest key); 8-bit radix passes over the keys find
// the key T of the keep-th largest row and how many rows of key T stay (those of the lowest
// slots).  Attention does not depend on the order of rows, so nothing is shifted: the i-th slot
// below `keep` that became free takes the i-th kept row behind it.  Sources (slots >= keep) and
// destinations (slots < keep) are disjoint, so the moves need no order among them.
//
// What bounds it is latency: a pass is a shared-memory histogram, a cluster barrier and a scan.
// So the keys are read once and stay in registers (slot order is warp, item, lane: a scan over
// all slots is one ballot per item and one sum over warps), every pass has one cluster barrier,
// and the passes end as soon as a digit's rows all stay.  8 x 2 heads of 4160 rows to 4096: 9.4 us;
// 16 x 2 of 32749 to 2048: 22 us, of which 12 bytes a row are 2 us of HBM time.
#include <cooperative_groups.h>

#include "common.cuh"
#include "kv4.cuh"
#include "runtime.cuh"

namespace cg = cooperative_groups;

namespace vx {
namespace {

constexpr int EV_THREADS = 512, EV_WARPS = EV_THREADS / 32;
constexpr int EV_MAX_CLUSTER = 16;  // above 8: not portable, but within one GPC of a B200
constexpr int EV_MAX_ITEMS = 16;  // keys of a thread
constexpr int EV_MAX_LEN = EV_THREADS * EV_MAX_CLUSTER * EV_MAX_ITEMS;  // 131072
static_assert(EV_MAX_LEN == 131072, "the length that the header names");
static_assert(EV_MAX_CLUSTER == 16, "the halves of the unrolled sums");

struct EvictArgs {
  uint8_t *k_codes, *k_scales, *v_codes, *v_scales;
  const float* weights;
  const int64_t* positions;
  float* weights_out;
  int64_t* positions_out;
  const int *lens, *seen;
  int* lens_out;
  int B, nkv, d, cap, max_len, keep, sink, recent;
  int* err;
};

// Rank of a row: larger weight, larger key; -0 counts as 0 and a NaN as the largest weight.
__device__ __forceinline__ uint32_t weight_key(float w) {
  const uint32_t u = __float_as_uint(w + 0.f);
  if (w != w) return 0xfffffffeu;
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

struct EvictShared {
  alignas(16) uint32_t hist[3][256], tot[256];
  uint32_t warp_n[2][EV_WARPS];
  uint32_t eq, holes, movers;  // of this block; read by the cluster
};

// Sum over the warps before this one and over all, of a value that each warp has put in n[].
__device__ __forceinline__ uint32_t warps_before(const uint32_t* n, int warp, uint32_t* all) {
  const int lane = threadIdx.x & 31;
  const uint32_t v = lane < EV_WARPS ? n[lane] : 0;
  *all = __reduce_add_sync(0xffffffffu, v);
  return __reduce_add_sync(0xffffffffu, lane < warp ? v : 0);
}

// n pieces of a type from one place to another, dealt to the block's threads.
template <class T, class Where>
__device__ __forceinline__ void move_pieces(uint32_t n, int tid, Where where) {
  constexpr int U = 4;
  for (uint32_t p0 = tid; p0 < n; p0 += U * EV_THREADS) {
    T x[U];
    T* onto[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t p = p0 + u * EV_THREADS;
      onto[u] = nullptr;
      if (p < n) {
        const T* from;
        where(p, &from, &onto[u]);
        x[u] = *from;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (onto[u]) *onto[u] = x[u];
  }
}

template <int ITEMS>
__global__ void __launch_bounds__(EV_THREADS, 2) kv4_evict_kernel(const EvictArgs a) {
  extern __shared__ __align__(16) uint32_t list[];  // free slots from the front, movers from the back
  uint32_t* to = list + EV_THREADS * ITEMS;         // the slots that this block's movers take
  __shared__ EvictShared s;
  cg::cluster_group cl = cg::this_cluster();
  const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  const int unit = blockIdx.x / C, b = unit / a.nkv, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int n = a.lens[b];
  const size_t row0 = (size_t)unit * a.cap;
  const bool first = unit % a.nkv == 0 && rank == 0 && tid == 0;
  if (n < 0 || n > a.max_len) {  // the same for every block of the cluster
    if (first) {
      record_error(a.err, VX_DEVICE_ERR_BOUNDS);
      a.lens_out[b] = n;
    }
    return;
  }
  if (first) a.lens_out[b] = min(n, a.keep);
  if (a.keep == 0) return;  // every row goes
  if (n <= a.keep) {        // every row stays
    for (int j = rank * EV_THREADS + tid; j < n; j += C * EV_THREADS) {
      if (a.weights_out != a.weights) a.weights_out[row0 + j] = a.weights[row0 + j];
      if (a.positions_out != a.positions) a.positions_out[row0 + j] = a.positions[row0 + j];
    }
    return;
  }
  const int base = (rank * EV_WARPS + warp) * 32 * ITEMS + lane;  // slot of item i: base + 32 i
  const int64_t since = (int64_t)a.seen[b] - a.recent;
  constexpr int G = ITEMS < 8 ? ITEMS : 8;  // rows of a thread that are on their way together
  uint32_t key[ITEMS];
#pragma unroll
  for (int i0 = 0; i0 < ITEMS; i0 += G) {
    float w[G];
    int64_t pos[G];
#pragma unroll
    for (int i = 0; i < G; ++i) {
      const int j = min(base + 32 * (i0 + i), n - 1);
      w[i] = a.weights[row0 + j];
      pos[i] = a.positions[row0 + j];
    }
#pragma unroll
    for (int i = 0; i < G; ++i)
      key[i0 + i] = base + 32 * (i0 + i) >= n ? 0 : pos[i] < a.sink || pos[i] >= since ? 0xffffffffu : weight_key(w[i]);
  }
  if (tid < 256) s.hist[0][tid] = 0;
  __syncthreads();
  uint32_t T = 0, left = (uint32_t)a.keep;  // rows still to be found among the keys that begin like T
  bool all_stay = false;                    // every key of T's digits so far stays
  for (int shift = 24, p = 0; shift >= 0 && !all_stay; shift -= 8, ++p) {
    uint32_t* h = s.hist[p % 3];
    if (tid < 256) s.hist[(p + 1) % 3][tid] = 0;  // last read two passes ago
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      if (base + 32 * i < n && (shift == 24 || ((key[i] ^ T) >> (shift + 8)) == 0))
        atomicAdd(&h[(key[i] >> shift) & 255], 1u);
    }
    cl.sync();
    if (tid < 128) {
      // unconditional loads of two counts, all on their way together: a round trip for four or eight
      // blocks (loads of one count: 32 units of 32749 rows 23.1 instead of 21.9 us)
      uint2 t = make_uint2(0, 0), v[8];
      auto at = [&](int r) { return reinterpret_cast<const uint2*>(cl.map_shared_rank(h, r))[tid]; };
      auto add = [&](const uint2& x) { t.x += x.x, t.y += x.y; };
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = at(min(r, C - 1));
      if (C > 4) {
#pragma unroll
        for (int r = 4; r < 8; ++r) v[r] = at(r);
#pragma unroll
        for (int r = 4; r < 8; ++r) add(v[r]);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (r < C) add(v[r]);
      if (C > 8) {
#pragma unroll
        for (int r = 0; r < 8; ++r) v[r] = at(r + 8);
#pragma unroll
        for (int r = 0; r < 8; ++r) add(v[r]);
      }
      reinterpret_cast<uint2*>(s.tot)[tid] = t;
    }
    __syncthreads();
    // every warp finds the digit at which the count from above reaches `left`
    uint32_t v[8], sum = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) sum += v[e] = s.tot[255 - (lane * 8 + e)];
    uint32_t incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t t = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += t;
    }
    const uint32_t hit = __ballot_sync(0xffffffffu, incl >= left);
    const int at = __ffs(hit) - 1;
    uint32_t above = incl - sum, digit = 255 - lane * 8, cnt = v[0];
#pragma unroll
    for (int e = 0; e < 7; ++e)
      if (above + v[e] < left && digit == (uint32_t)(255 - lane * 8 - e)) {
        above += v[e];
        --digit;
        cnt = v[e + 1];
      }
    above = __shfl_sync(0xffffffffu, above, at);
    digit = __shfl_sync(0xffffffffu, digit, at);
    cnt = __shfl_sync(0xffffffffu, cnt, at);
    left -= above;
    T |= digit << shift;
    all_stay = cnt == left;
    __syncthreads();  // tot is read
  }

  // rows of key T that stay: all of them, or the first `left` in slot order
  uint32_t eq_before = 0;
  if (!all_stay) {
    uint32_t c = 0;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) c += __popc(__ballot_sync(0xffffffffu, base + 32 * i < n && key[i] == T));
    if (lane == 0) s.warp_n[0][warp] = c;
    __syncthreads();
    uint32_t all;
    eq_before = warps_before(s.warp_n[0], warp, &all);
    if (tid == 0) s.eq = all;
    cl.sync();
    const uint32_t e = lane < rank ? *cl.map_shared_rank(&s.eq, lane) : 0;
    eq_before += __reduce_add_sync(0xffffffffu, e);
  }
  const uint32_t below = (1u << lane) - 1;
  uint32_t stays = 0, holes = 0, movers = 0;  // bit i: item i; counts of this warp
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int j = base + 32 * i;
    bool keep = j < n && key[i] >= T;
    if (!all_stay) {
      const bool eq = j < n && key[i] == T;
      const uint32_t m = __ballot_sync(0xffffffffu, eq);
      if (eq) keep = eq_before + __popc(m & below) < left;
      eq_before += __popc(m);
    }
    stays |= (uint32_t)keep << i;
    holes += __popc(__ballot_sync(0xffffffffu, j < n && j < a.keep && !keep));
    movers += __popc(__ballot_sync(0xffffffffu, j >= a.keep && keep));
  }
  if (lane == 0) s.warp_n[1][warp] = holes | movers << 16;  // at most 16384 each in a block
  __syncthreads();
  uint32_t all;
  const uint32_t before = warps_before(s.warp_n[1], warp, &all);
  if (tid == 0) {
    s.holes = all & 0xffff;
    s.movers = all >> 16;
  }
  uint32_t hb = before & 0xffff, mb = before >> 16;
  constexpr int kLast = EV_THREADS * ITEMS - 1;
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int j = base + 32 * i;
    const bool keep = stays >> i & 1, hole = j < n && j < a.keep && !keep, mover = j >= a.keep && keep;
    const uint32_t hm = __ballot_sync(0xffffffffu, hole), mm = __ballot_sync(0xffffffffu, mover);
    if (hole) list[hb + __popc(hm & below)] = j;
    if (mover) list[kLast - (mb + __popc(mm & below))] = j;
    hb += __popc(hm);
    mb += __popc(mm);
  }
  // rows that stay where they are: loads of eight at a time, ahead of the stores that may alias them
  const bool apart = a.weights_out != a.weights || a.positions_out != a.positions;
  if (apart && (rank * EV_WARPS + warp) * 32 * ITEMS < a.keep) {
#pragma unroll
    for (int i0 = 0; i0 < ITEMS; i0 += G) {
      float w[G];
      int64_t pos[G];
#pragma unroll
      for (int i = 0; i < G; ++i) {
        const int j = base + 32 * (i0 + i);
        if ((stays >> (i0 + i) & 1) && j < a.keep) w[i] = a.weights[row0 + j], pos[i] = a.positions[row0 + j];
      }
#pragma unroll
      for (int i = 0; i < G; ++i) {
        const int j = base + 32 * (i0 + i);
        if ((stays >> (i0 + i) & 1) && j < a.keep) a.weights_out[row0 + j] = w[i], a.positions_out[row0 + j] = pos[i];
      }
    }
  }
  cl.sync();
  // lane r: free slots and movers of the blocks before block r
  const uint32_t h_r = lane < C ? *cl.map_shared_rank(&s.holes, lane) : 0;
  const uint32_t m0 = __reduce_add_sync(0xffffffffu, lane < rank ? *cl.map_shared_rank(&s.movers, lane) : 0);
  uint32_t hole0 = h_r;
#pragma unroll
  for (int o = 1; o < EV_MAX_CLUSTER; o <<= 1) {
    const uint32_t t = __shfl_up_sync(0xffffffffu, hole0, o);
    if (lane >= o) hole0 += t;
  }
  hole0 -= h_r;
  const uint32_t mine = all >> 16;
  // where each mover goes: the block that holds the g-th free slot is the last one whose first is not above g
  uint32_t first_of[EV_MAX_CLUSTER];
#pragma unroll
  for (int r = 0; r < EV_MAX_CLUSTER; ++r) first_of[r] = r < C ? __shfl_sync(0xffffffffu, hole0, r) : 0xffffffffu;
  for (uint32_t i = tid; i < mine; i += EV_THREADS) {
    const uint32_t g = m0 + i;
    int owner = 0;
    uint32_t start = 0;
#pragma unroll
    for (int r = 1; r < EV_MAX_CLUSTER; ++r)
      if (r < C && g >= first_of[r]) owner = r, start = first_of[r];
    to[i] = cl.map_shared_rank(list, owner)[g - start];
  }
  __syncthreads();
  // one kind of piece after the other, each with full warps and four loads of a thread in flight
  auto src = [&](uint32_t i) { return row0 + list[kLast - i]; };
  auto dst = [&](uint32_t i) { return row0 + to[i]; };
  const int cb = a.d / 32;             // 16-byte pieces of a row's codes of K: 4 or 2
  const int lg = a.d == 128 ? 2 : 1;  // words of a row's scales of K and V: 4 or 2
  move_pieces<uint4>(mine << (lg + 1), tid, [&](uint32_t p, const uint4** from, uint4** onto) {
    const uint32_t i = p >> (lg + 1), c = p & (2 * cb - 1);
    uint8_t* base = c < (uint32_t)cb ? a.k_codes : a.v_codes;
    const size_t off = (size_t)(c & (cb - 1)) * 16;
    *from = reinterpret_cast<const uint4*>(base + src(i) * (a.d / 2) + off);
    *onto = reinterpret_cast<uint4*>(base + dst(i) * (a.d / 2) + off);
  });
  move_pieces<uint32_t>(mine << lg, tid, [&](uint32_t p, const uint32_t** from, uint32_t** onto) {
    const uint32_t i = p >> lg, c = p & ((1 << lg) - 1), words = 1u << (lg - 1);
    uint8_t* base = c < words ? a.k_scales : a.v_scales;
    const size_t off = (size_t)(c & (words - 1)) * 4;
    *from = reinterpret_cast<const uint32_t*>(base + src(i) * (a.d / 16) + off);
    *onto = reinterpret_cast<uint32_t*>(base + dst(i) * (a.d / 16) + off);
  });
  move_pieces<float>(mine, tid, [&](uint32_t i, const float** from, float** onto) {
    *from = a.weights + src(i);
    *onto = a.weights_out + dst(i);
  });
  move_pieces<int64_t>(mine, tid, [&](uint32_t i, const int64_t** from, int64_t** onto) {
    *from = a.positions + src(i);
    *onto = a.positions_out + dst(i);
  });
  cl.sync();  // the lists are read by the other blocks
}

// Blocks of a cluster and keys of a thread.  More blocks scan faster, but clusters of 8 and more cost
// more to launch and to bring together, the more so where several share a GPC.  So they double while a
// thread would have more than 4 keys (from 4 to 8 blocks: 5) and the blocks are few: two to an SM, for
// 16 in a cluster one (16 units of 4160 rows: 4 blocks 10.4 us, 8 14.1; of 16000: 4 29.0, 8 25.0, 16
// 43.0; 32 units of 32749: 4 36.2, 8 28.6, 16 62.2; 64 units of 16000: 2 46.2, 4 34.9, 8 45.7).  The
// keys of a thread are as few as hold the longest sequence.
void evict_shape(int units, int max_len, int* C, int* items) {
  *C = 1;
  while (*C < EV_MAX_CLUSTER && max_len > EV_THREADS * (*C == 4 ? 5 : 4) * *C &&
         (long long)units * *C * 2 <= (*C < 8 ? 296 : 148))
    *C *= 2;
  while (max_len > EV_THREADS * EV_MAX_ITEMS * *C) *C *= 2;
  *items = 2;
  while (max_len > EV_THREADS * *items * *C) *items *= 2;
}

template <int ITEMS>
cudaError_t evict_launch(cudaLaunchConfig_t& cfg, const EvictArgs& a) {
  cfg.dynamicSmemBytes = (size_t)EV_THREADS * ITEMS * 8;
  return cudaLaunchKernelEx(&cfg, kv4_evict_kernel<ITEMS>, a);
}

}  // namespace

template <int ITEMS>
static cudaError_t evict_allow() {
  const cudaError_t e = cudaFuncSetAttribute(kv4_evict_kernel<ITEMS>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             EV_THREADS * ITEMS * 8);
  if (e != cudaSuccess) return e;
  return cudaFuncSetAttribute(kv4_evict_kernel<ITEMS>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
}

cudaError_t kv4_evict_configure() {
  cudaError_t e = evict_allow<2>();
  if (e == cudaSuccess) e = evict_allow<4>();
  if (e == cudaSuccess) e = evict_allow<8>();
  if (e == cudaSuccess) e = evict_allow<16>();
  return e;
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
  if (lens_out == lens || lens_out == seen)
    return fail(ctx, VX_ERR_ARG, "kv4_evict: lens_out must be neither lens nor seen");
  if (max_len < 0 || max_len > c->capacity)
    return fail(ctx, VX_ERR_SHAPE, "kv4_evict: max_len %d outside 0..%d", max_len, c->capacity);
  if (max_len > EV_MAX_LEN) return fail(ctx, VX_ERR_SHAPE, "kv4_evict: max_len %d > %d", max_len, EV_MAX_LEN);
  if (keep < 0 || sink < 0 || recent < 0 || (long long)sink + recent > keep)
    return fail(ctx, VX_ERR_SHAPE, "kv4_evict: sink %d + recent %d must fit in keep %d", sink, recent, keep);
  DeviceGuard guard(ctx->device);
  EvictArgs a = {c->k_codes, c->k_scales, c->v_codes, c->v_scales, c->weights, c->positions, weights_out,
                 positions_out, lens, seen, lens_out, c->batch, c->n_kv_heads, c->head_dim, c->capacity, max_len, keep,
                 sink, recent, ctx->dev_err};
  int C, items;
  evict_shape(c->batch * c->n_kv_heads, max_len, &C, &items);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(c->batch * c->n_kv_heads * C);
  cfg.blockDim = dim3(EV_THREADS);
  cfg.stream = pick_stream(ctx, stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  count_launch();
  VX_CUDA(ctx, items == 2    ? evict_launch<2>(cfg, a)
               : items == 4  ? evict_launch<4>(cfg, a)
               : items == 8  ? evict_launch<8>(cfg, a)
                             : evict_launch<16>(cfg, a));
  return VX_OK;
}
