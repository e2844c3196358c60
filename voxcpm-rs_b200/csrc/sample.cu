// Token sampling from logits (vx_sample): temperature, top-k, top-p, min-p and a draw from a
// given random number, one cluster of C thread blocks per row of logits, the row in their shared
// memory.
//
// A token's weight is w = rint(exp((l - lmax) / T) * 2^44) as a 64-bit integer: sums of weights
// are exact whatever their order (a row of 2^18 tokens stays below 2^62), so every block and
// every order of atomics finds the same border.  The tokens that stay are a prefix of the order
// (logit descending, index ascending), described by the key of its last logit and how many
// tokens of that key stay; radix passes over the ordered keys find it, by count for top-k, by
// weight for top-p.  The draw takes the first token in index order whose running sum of staying
// weights exceeds u * total.
#include <cooperative_groups.h>

#include <cfloat>

#include "common.cuh"
#include "runtime.cuh"

namespace cg = cooperative_groups;

namespace vx {
namespace {

typedef unsigned long long u64;

constexpr int SP_THREADS = 1024;
constexpr int SP_MAX_CLUSTER = 8;
constexpr int SP_SLICE = 32768;       // logits of a block: 128 KB
constexpr int SP_MAX_VOCAB = 1 << 18;
constexpr double SP_ONE = 17592186044416.0;  // 2^44

struct SampleArgs {
  const float* logits;
  long long ld;
  int rows, vocab, slice;
  const float *u, *temperature;
  const int* top_k;
  const float *top_p, *min_p;
  int* ids;
  float* logprob;
};

// ascending with the logit; -0 and 0 are the same
__device__ __forceinline__ uint32_t key_of(float l) {
  const uint32_t u = __float_as_uint(l + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float logit_of(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

__device__ __forceinline__ u64 weight_of(float l, float lmax, double T) {
  if (l == lmax) return (u64)SP_ONE;
  const double z = ((double)l - (double)lmax) / T;
  // below exp(-31.2) 2^44 = 1/2 a weight is 0; so is that of -inf (or anything next to +inf) at T = inf, a NaN here
  return z > -31.5 ? __double2ull_rn(exp(z) * SP_ONE) : 0;
}

__device__ __forceinline__ u64 warp_sum64(u64 v) {
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

struct SampleShared {
  u64 mass[2][256], tot[256];
  u64 warp64[32], part64[2];
  uint32_t warp32[32], part32[4];
  u64 left;
  uint32_t prefix;
  float fmax;
  int bad;
};

// Block-wide sums; every thread gets the total.
__device__ __forceinline__ u64 block_sum64(u64 v, u64* red) {
  v = warp_sum64(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  u64 t = 0;
  for (int w = 0; w < SP_THREADS / 32; ++w) t += red[w];
  return t;
}

// The largest key T with sum(value of tokens with key >= T) >= need; *left = need minus the sum
// of those above T.  value(key) is summed over this cluster's tokens.
template <class F>
__device__ uint32_t radix_find(cg::cluster_group& cl, SampleShared& s, const float* x, int cnt, u64 need, u64* left,
                               F value) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, C = (int)cl.num_blocks();
  uint32_t prefix = 0;
  for (int pass = 0; pass < 4; ++pass) {
    const int shift = 24 - 8 * pass;
    u64* h = s.mass[pass & 1];
    cl.sync();  // every block is done with what it read of the pass before last
    if (tid < 256) h[tid] = 0;
    __syncthreads();
    for (int j = tid; j < cnt; j += SP_THREADS) {
      const uint32_t k = key_of(x[j]);
      if (pass == 0 || (k >> (shift + 8)) == (prefix >> (shift + 8))) {
        const u64 v = value(x[j], k);
        if (v) atomicAdd(&h[(k >> shift) & 255], v);
      }
    }
    cl.sync();
    if (tid < 256) {
      u64 t = 0;
      for (int r = 0; r < C; ++r) t += cl.map_shared_rank(h, r)[tid];
      s.tot[tid] = t;
    }
    __syncthreads();
    if (warp == 0) {
      u64 v[8], sum = 0;
      for (int e = 0; e < 8; ++e) sum += v[e] = s.tot[255 - (lane * 8 + e)];
      u64 incl = sum;
      for (int o = 1; o < 32; o <<= 1) {
        const u64 t = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += t;
      }
      u64 above = incl - sum;
      if (above < need && incl >= need) {
        int e = 0;
        while (above + v[e] < need) above += v[e++];
        s.prefix = prefix | ((uint32_t)(255 - (lane * 8 + e)) << shift);
        s.left = need - above;
      }
    }
    __syncthreads();
    prefix = s.prefix;
    need = s.left;
  }
  *left = need;
  return prefix;
}

__global__ void __launch_bounds__(SP_THREADS) sample_kernel(const SampleArgs a) {
  extern __shared__ __align__(16) float x[];
  __shared__ SampleShared s;
  cg::cluster_group cl = cg::this_cluster();
  const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  const int row = blockIdx.x / C, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const float* src = a.logits + (size_t)row * a.ld;
  const int lo = min(a.vocab, rank * a.slice), cnt = min(a.vocab, lo + a.slice) - lo;

  float m = -INFINITY;
  int bad = 0;
  for (int j = tid; j < cnt; j += SP_THREADS) {
    const float l = __ldg(src + lo + j);
    x[j] = l;
    m = fmaxf(m, l);
    bad |= l != l;
  }
  m = warp_max(m);
  bad = __any_sync(0xffffffffu, bad);
  if (lane == 0) {
    s.warp32[warp] = __float_as_uint(m);
    if (warp == 0) s.bad = 0;
  }
  __syncthreads();
  if (lane == 0 && bad) s.bad = 1;
  if (tid == 0) {
    for (int w = 1; w < SP_THREADS / 32; ++w) m = fmaxf(m, __uint_as_float(s.warp32[w]));
    s.fmax = m;
  }
  cl.sync();
  float lmax = -INFINITY;
  bad = 0;
  for (int r = 0; r < C; ++r) {
    lmax = fmaxf(lmax, *cl.map_shared_rank(&s.fmax, r));
    bad |= *cl.map_shared_rank(&s.bad, r);
  }
  const float temp = a.temperature ? a.temperature[row] : 1.f;
  const bool greedy = temp == 0.f;
  const bool none = bad || lmax == -INFINITY || !(temp >= 0.f);
  if (none) {  // the same for the whole cluster
    if (rank == 0 && tid == 0) {
      a.ids[row] = -1;
      if (a.logprob) a.logprob[row] = bad || !(temp >= 0.f) ? NAN : -INFINITY;
    }
    cl.sync();  // fmax and bad are read by the other blocks
    return;
  }
  const double T = greedy ? 1.0 : (double)temp;
  int k = a.top_k ? a.top_k[row] : 0;
  if (greedy) k = 1;
  uint32_t Tk = 0, ties = 0xffffffffu;  // tokens with key > Tk stay, and the first `ties` of key Tk
  if (k > 0 && k < a.vocab) {
    u64 left;
    Tk = radix_find(cl, s, x, cnt, (u64)k, &left, [](float, uint32_t) { return (u64)1; });
    ties = (uint32_t)left;
  }
  const float p = a.top_p ? a.top_p[row] : 1.f;
  if (p < 1.f) {
    const u64 wt = ties == 0xffffffffu ? 0 : weight_of(logit_of(Tk), lmax, T);
    u64 mass = 0;
    for (int j = tid; j < cnt; j += SP_THREADS)
      if (key_of(x[j]) > Tk || ties == 0xffffffffu) mass += weight_of(x[j], lmax, T);
    mass = block_sum64(mass, s.warp64);
    if (tid == 0) s.part64[0] = mass;
    cl.sync();
    mass = ties == 0xffffffffu ? 0 : ties * wt;
    for (int r = 0; r < C; ++r) mass += *cl.map_shared_rank(&s.part64[0], r);
    const double want = ceil((double)p * (double)mass);
    const u64 need = want < 1.0 ? 1 : (u64)want;
    const uint32_t Tk0 = Tk, ties0 = ties;
    const u64 above = mass - (ties0 == 0xffffffffu ? 0 : ties0 * wt);
    if (ties0 == 0xffffffffu || need <= above) {
      u64 left;
      Tk = radix_find(cl, s, x, cnt, need, &left, [&](float l, uint32_t key) {
        return key > Tk0 || ties0 == 0xffffffffu ? weight_of(l, lmax, T) : (u64)0;
      });
      const u64 w = weight_of(logit_of(Tk), lmax, T);
      ties = (uint32_t)((left + w - 1) / w);
    } else {
      ties = (uint32_t)((need - above + wt - 1) / wt);
    }
  }
  double least = a.min_p ? fmin((double)a.min_p[row], 1.0) * SP_ONE : 0.0;
  if (!(least >= 0.0)) least = 0.0;

  // which tokens of key Tk stay: the first `ties` in index order
  uint32_t eq_base = 0;
  if (ties != 0xffffffffu) {
    uint32_t c = 0;
    for (int j = tid; j < cnt; j += SP_THREADS) c += key_of(x[j]) == Tk;
    const u64 t = block_sum64(c, s.warp64);
    if (tid == 0) s.part32[0] = (uint32_t)t;
    cl.sync();
    for (int r = 0; r < rank; ++r) eq_base += *cl.map_shared_rank(&s.part32[0], r);
  }
  // weight of every staying token, chunk by chunk in index order; the sum of this block
  auto chunk_weight = [&](int j0, uint32_t& base) {
    const int j = j0 + tid;
    const bool in = j < cnt;
    const float l = in ? x[j] : -INFINITY;
    const uint32_t key = key_of(l);
    bool stays = in;
    if (ties != 0xffffffffu) {
      const uint32_t eq = __ballot_sync(0xffffffffu, in && key == Tk);
      __syncthreads();
      if (lane == 0) s.warp32[warp] = __popc(eq);
      __syncthreads();
      uint32_t before = 0, all = 0;
      for (int w = 0; w < 32; ++w) {
        if (w < warp) before += s.warp32[w];
        all += s.warp32[w];
      }
      stays = in && (key > Tk || (key == Tk && base + before + __popc(eq & ((1u << lane) - 1)) < ties));
      base += all;
    }
    if (!stays) return (u64)0;
    const u64 w = weight_of(l, lmax, T);
    return (double)w >= least ? w : (u64)0;
  };
  u64 sum = 0;
  uint32_t base = eq_base;
  for (int j0 = 0; j0 < cnt; j0 += SP_THREADS) sum += chunk_weight(j0, base);
  sum = block_sum64(sum, s.warp64);
  if (tid == 0) s.part64[1] = sum;
  cl.sync();
  u64 total = 0, before = 0;
  for (int r = 0; r < C; ++r) {
    const u64 t = *cl.map_shared_rank(&s.part64[1], r);
    if (r < rank) before += t;
    total += t;
  }
  const float uf = a.u[row];
  const double ud = uf > 0.f ? (double)uf : 0.0;
  const double at_d = floor(ud * (double)total);
  const u64 at = at_d >= (double)total ? total - 1 : (u64)at_d < total ? (u64)at_d : total - 1;
  if (before <= at && at < before + sum) {  // this block holds the token
    base = eq_base;
    u64 run = before;
    for (int j0 = 0; j0 < cnt; j0 += SP_THREADS) {
      const u64 w = chunk_weight(j0, base);
      u64 incl = w;
      for (int o = 1; o < 32; o <<= 1) {
        const u64 t = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += t;
      }
      __syncthreads();
      if (lane == 31) s.warp64[warp] = incl;
      __syncthreads();
      u64 wb = run, all = 0;
      for (int q = 0; q < 32; ++q) {
        if (q < warp) wb += s.warp64[q];
        all += s.warp64[q];
      }
      if (wb + incl - w <= at && at < wb + incl) {
        a.ids[row] = lo + j0 + tid;
        if (a.logprob) a.logprob[row] = (float)log((double)w / (double)total);
      }
      run += all;
      if (run > at) break;
    }
  }
  cl.sync();  // part64 is read by the other blocks
}

int cluster_of(int rows, int vocab) {
  int c = 1;
  while (c < SP_MAX_CLUSTER && (vocab > SP_SLICE * c || (rows * c < 148 && vocab > 4096 * c))) c *= 2;
  return c;
}

}  // namespace

cudaError_t sample_configure() {
  return cudaFuncSetAttribute(sample_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SP_SLICE * 4);
}

}  // namespace vx

using namespace vx;

extern "C" int vx_sample(vx_ctx* ctx, const float* logits, int64_t row_stride, int rows, int vocab, const float* u,
                         const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                         int32_t* ids, float* logprob, vx_stream stream) {
  if (!ctx || !logits || !u || !ids) return VX_ERR_ARG;
  if (rows < 0 || rows > (1 << 20)) return fail(ctx, VX_ERR_SHAPE, "sample: %d rows outside 0..2^20", rows);
  if (vocab <= 0 || vocab > SP_MAX_VOCAB)
    return fail(ctx, VX_ERR_SHAPE, "sample: vocabulary %d outside 1..%d", vocab, SP_MAX_VOCAB);
  if (row_stride < vocab) return fail(ctx, VX_ERR_SHAPE, "sample: row stride below the vocabulary");
  if (rows == 0) return VX_OK;
  DeviceGuard guard(ctx->device);
  const int C = cluster_of(rows, vocab);
  SampleArgs a = {logits, row_stride, rows, vocab, (vocab + C - 1) / C, u, temperature, top_k, top_p, min_p, ids,
                  logprob};
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(rows * C);
  cfg.blockDim = dim3(SP_THREADS);
  cfg.dynamicSmemBytes = (size_t)a.slice * 4;
  cfg.stream = pick_stream(ctx, stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  count_launch();
  VX_CUDA(ctx, cudaLaunchKernelEx(&cfg, sample_kernel, a));
  return VX_OK;
}
