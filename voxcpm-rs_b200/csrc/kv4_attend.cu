// Decode attention over the 4-bit KV cache (vx_kv4_attend): one query token of each sequence
// against its cached rows, s_j = scale * q . k_j, p = softmax(s), out = sum_j p_j v_j, and with
// `track` the running weight of a row += the sum of p_j over the query heads that share it.
//
// kv4_split_kernel: grid (splits, B * nkv * head blocks of up to 8 query heads); a split covers
// a run of positions and leaves (m, l, o) of its heads, or the result where there is one split.
// kv4_finish_kernel: merges the splits, and turns the scores that a tracking call left in the
// workspace into weights once the maxima and sums over all splits are known.
#include <cfloat>

#include "common.cuh"
#include "kv4.cuh"
#include "runtime.cuh"

namespace vx {
namespace {

constexpr int HB = 8;  // query heads of a block

struct AttendArgs {
  const float* q;
  long long ldq;
  const uint8_t *k_codes, *k_scales, *v_codes, *v_scales;
  const int* lens;
  float* weights;
  float* out;
  long long ldo;
  float scale;  // of the scores, times log2(e)
  int B, nkv, nrep, nhb, cap, max_len, chunk, nsplit;
  float* scores;  // [B * nkv * nhb][max_len][8], base-2 scores of a tracking call
  float* part_ml; // [B * nkv * nhb][nsplit][8][2]
  float* part_o;  // [B * nkv * nhb][nsplit][8][d]
  int* err;
};

// length of sequence b, -1 if it is out of range
__device__ __forceinline__ int seq_len(const AttendArgs& a, int b) {
  const int n = a.lens[b];
  return n < 0 || n > a.max_len ? -1 : n;
}

template <int D>
__global__ void __launch_bounds__(256) kv4_split_kernel(const AttendArgs a) {
  const int unit = blockIdx.y, split = blockIdx.x;
  const int hb = unit % a.nhb, g = (unit / a.nhb) % a.nkv, b = unit / (a.nhb * a.nkv);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int head = hb * HB + warp;
  const int n = seq_len(a, b);
  constexpr int DPL = D / 32;
  float* out = a.out + (size_t)b * a.ldo + (size_t)(g * a.nrep + head) * D + lane * DPL;
  if (n <= 0) {
    if (n < 0 && threadIdx.x == 0) record_error(a.err, VX_DEVICE_ERR_BOUNDS);
    if (split == 0 && head < a.nrep)
      for (int e = 0; e < DPL; ++e) out[e] = n < 0 ? NAN : 0.f;
    return;
  }
  const int j0 = split * a.chunk, j1 = min(n, j0 + a.chunk);
  if (j0 >= j1 || head >= a.nrep) return;
  const size_t row0 = (size_t)(b * a.nkv + g) * a.cap;
  float q[DPL], o[DPL];
  for (int e = 0; e < DPL; ++e) {
    q[e] = a.q[(size_t)b * a.ldq + (size_t)(g * a.nrep + head) * D + lane * DPL + e];
    o[e] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  auto load = [&](const uint8_t* codes, const uint8_t* scales, int j, float* x) {
    const float sc = e4m3_to_f32(scales[(row0 + j) * (D / KV4_GROUP) + lane * DPL / KV4_GROUP]);
    for (int e = 0; e < DPL; e += 2) {
      const uint32_t h = e2m1x2_to_h2(codes[(row0 + j) * (D / 2) + (lane * DPL + e) / 2]);
      x[e] = h2_lo(h) * sc;
      x[e + 1] = h2_hi(h) * sc;
    }
  };
  for (int j = j0; j < j1; ++j) {
    float x[DPL], s = 0.f;
    load(a.k_codes, a.k_scales, j, x);
    for (int e = 0; e < DPL; ++e) s = fmaf(q[e], x[e], s);
    s = warp_sum(s) * a.scale;
    if (a.scores && lane == 0) a.scores[((size_t)unit * a.max_len + j) * HB + warp] = s;
    const float mn = fmaxf(m, s);
    const float alpha = m == mn ? 1.f : exp2f(m - mn), p = exp2f(s - mn);
    l = l * alpha + p;
    load(a.v_codes, a.v_scales, j, x);
    for (int e = 0; e < DPL; ++e) o[e] = fmaf(p, x[e], o[e] * alpha);
    m = mn;
  }
  if (a.nsplit == 1) {
    for (int e = 0; e < DPL; ++e) out[e] = o[e] / l;
  } else {
    float* po = a.part_o + (((size_t)unit * a.nsplit + split) * HB + warp) * D + lane * DPL;
    for (int e = 0; e < DPL; ++e) po[e] = o[e];
  }
  if (a.part_ml && lane == 0) {
    float* p = a.part_ml + (((size_t)unit * a.nsplit + split) * HB + warp) * 2;
    p[0] = m;
    p[1] = l;
  }
}

// Maximum and 1 / sum of one head over the active splits, by one warp.
__device__ __forceinline__ void head_stats(const AttendArgs& a, int unit, int r, int active, float* M, float* inv) {
  const int lane = threadIdx.x & 31;
  const float* p = a.part_ml + ((size_t)unit * a.nsplit * HB + r) * 2;
  float m = -INFINITY, l = 0.f;
  for (int s = lane; s < active; s += 32) m = fmaxf(m, p[(size_t)s * HB * 2]);
  m = warp_max(m);
  for (int s = lane; s < active; s += 32) l += p[(size_t)s * HB * 2 + 1] * exp2f(p[(size_t)s * HB * 2] - m);
  *M = m;
  *inv = 1.f / warp_sum(l);
}

// Blocks 0 .. units * 8 - 1 merge one head each (where there is more than one split); the blocks
// behind them add the probabilities of 256 positions of one KV head to its weights.
template <int D>
__global__ void __launch_bounds__(256) kv4_finish_kernel(const AttendArgs a, int merge_blocks, int chunks) {
  __shared__ float sm[64 * 2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if ((int)blockIdx.x < merge_blocks) {
    const int unit = blockIdx.x / HB, r = blockIdx.x % HB;
    const int hb = unit % a.nhb, g = (unit / a.nhb) % a.nkv, b = unit / (a.nhb * a.nkv);
    const int n = seq_len(a, b);
    if (n <= 0 || hb * HB + r >= a.nrep) return;
    const int active = (n + a.chunk - 1) / a.chunk;
    __shared__ float acc[8][D];
    float M, inv;
    head_stats(a, unit, r, active, &M, &inv);
    constexpr int DPL = D / 32;
    float o[DPL] = {};
    for (int s = warp; s < active; s += 8) {
      const float f = exp2f(a.part_ml[(((size_t)unit * a.nsplit + s) * HB + r) * 2] - M);
      const float* po = a.part_o + (((size_t)unit * a.nsplit + s) * HB + r) * D + lane * DPL;
      for (int e = 0; e < DPL; ++e) o[e] = fmaf(f, po[e], o[e]);
    }
    for (int e = 0; e < DPL; ++e) acc[warp][lane * DPL + e] = o[e];
    __syncthreads();
    if ((int)threadIdx.x < D) {
      float t = 0.f;
      for (int w = 0; w < 8; ++w) t += acc[w][threadIdx.x];
      a.out[(size_t)b * a.ldo + (size_t)(g * a.nrep + hb * HB + r) * D + threadIdx.x] = t * inv;
    }
    return;
  }
  const int i = blockIdx.x - merge_blocks;
  const int c = i % chunks, bg = i / chunks, b = bg / a.nkv;
  const int n = seq_len(a, b);
  if (n <= 0 || c * 256 >= n) return;
  const int active = (n + a.chunk - 1) / a.chunk;
  const int j = c * 256 + threadIdx.x;
  float w = 0.f;
  for (int hb = 0; hb < a.nhb; ++hb) {
    const int unit = bg * a.nhb + hb, heads = min(HB, a.nrep - hb * HB);
    __syncthreads();
    if (warp < heads) {
      float M, inv;
      head_stats(a, unit, warp, active, &M, &inv);
      if (lane == 0) {
        sm[warp * 2] = M;
        sm[warp * 2 + 1] = inv;
      }
    }
    __syncthreads();
    if (j < n) {
      const float* s = a.scores + ((size_t)unit * a.max_len + j) * HB;
      for (int r = 0; r < heads; ++r) w += exp2f(s[r] - sm[r * 2]) * sm[r * 2 + 1];
    }
  }
  if (j < n) a.weights[(size_t)bg * a.cap + j] += w;
}

struct AttendPlan {
  int nhb, chunk, nsplit;
  size_t ml_bytes, o_bytes, score_bytes;
};

AttendPlan plan_of(const vx_kv4* c, int nh, int max_len, int track) {
  AttendPlan p;
  const int nrep = nh / c->n_kv_heads;
  p.nhb = (nrep + HB - 1) / HB;
  const long long units = (long long)c->batch * c->n_kv_heads * p.nhb;
  long long chunk = (units * max_len + 148 * 8 - 1) / (148 * 8);
  chunk = std::min<long long>(2048, std::max<long long>(64, (chunk + 31) / 32 * 32));
  p.chunk = (int)chunk;
  p.nsplit = std::max(1, (int)((max_len + chunk - 1) / chunk));
  const bool parts = p.nsplit > 1 || track;
  p.ml_bytes = parts ? (size_t)units * p.nsplit * HB * 2 * 4 : 0;
  p.o_bytes = p.nsplit > 1 ? (size_t)units * p.nsplit * HB * c->head_dim * 4 : 0;
  p.score_bytes = track ? (size_t)units * max_len * HB * 4 : 0;
  return p;
}

}  // namespace

}  // namespace vx

using namespace vx;

extern "C" {

size_t vx_kv4_attend_workspace(const vx_kv4* c, int nh, int max_len, int track) {
  if (!c || c->n_kv_heads <= 0 || nh <= 0 || nh % c->n_kv_heads != 0 || max_len < 0 || c->batch <= 0) return 0;
  const AttendPlan p = plan_of(c, nh, max_len, track);
  return p.ml_bytes + p.o_bytes + p.score_bytes;
}

int vx_kv4_attend(vx_ctx* ctx, const vx_kv4* c, const float* q, int64_t q_stride, int nh, const int32_t* lens,
                  int max_len, float scale, int track, float* out, int64_t out_stride, void* workspace,
                  size_t workspace_bytes, vx_stream stream) {
  const int rc = kv4_check(ctx, c, "kv4_attend");
  if (rc) return rc;
  if (!q || !lens || !out) return fail(ctx, VX_ERR_ARG, "kv4_attend: q, lens and out are needed");
  if (nh <= 0 || nh % c->n_kv_heads != 0 || nh / c->n_kv_heads > 64)
    return fail(ctx, VX_ERR_SHAPE, "kv4_attend: %d query heads do not share %d KV heads (at most 64 each)", nh,
                c->n_kv_heads);
  if (max_len < 0 || max_len > c->capacity)
    return fail(ctx, VX_ERR_SHAPE, "kv4_attend: max_len %d outside 0..%d", max_len, c->capacity);
  if (track && !c->weights) return fail(ctx, VX_ERR_ARG, "kv4_attend: the cache keeps no weights to add to");
  if ((((uintptr_t)q | (uintptr_t)out) & 15) || q_stride % 4 != 0 || out_stride % 4 != 0 ||
      q_stride < (int64_t)nh * c->head_dim || out_stride < (int64_t)nh * c->head_dim)
    return fail(ctx, VX_ERR_ARG, "kv4_attend: q and out must be 16-byte aligned rows of nh * head_dim floats");
  const AttendPlan p = plan_of(c, nh, max_len, track);
  const size_t need = p.ml_bytes + p.o_bytes + p.score_bytes;
  if (need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15)))
    return fail(ctx, VX_ERR_ARG, "kv4_attend: %zu bytes of 16-byte aligned workspace are needed", need);
  DeviceGuard guard(ctx->device);
  cudaStream_t st = pick_stream(ctx, stream);
  char* ws = static_cast<char*>(workspace);
  AttendArgs a = {};
  a.q = q;
  a.ldq = q_stride;
  a.k_codes = c->k_codes;
  a.k_scales = c->k_scales;
  a.v_codes = c->v_codes;
  a.v_scales = c->v_scales;
  a.lens = lens;
  a.weights = track ? c->weights : nullptr;
  a.out = out;
  a.ldo = out_stride;
  a.scale = scale * KV4_LOG2E;
  a.B = c->batch;
  a.nkv = c->n_kv_heads;
  a.nrep = nh / c->n_kv_heads;
  a.nhb = p.nhb;
  a.cap = c->capacity;
  a.max_len = max_len;
  a.chunk = p.chunk;
  a.nsplit = p.nsplit;
  if (p.ml_bytes) a.part_ml = reinterpret_cast<float*>(ws);
  if (p.o_bytes) a.part_o = reinterpret_cast<float*>(ws + p.ml_bytes);
  if (p.score_bytes) a.scores = reinterpret_cast<float*>(ws + p.ml_bytes + p.o_bytes);
  a.err = ctx->dev_err;
  const int units = a.B * a.nkv * a.nhb;
  count_launch();
  if (c->head_dim == 128)
    kv4_split_kernel<128><<<dim3(p.nsplit, units), 256, 0, st>>>(a);
  else
    kv4_split_kernel<64><<<dim3(p.nsplit, units), 256, 0, st>>>(a);
  VX_CUDA(ctx, cudaGetLastError());
  if (!need || max_len == 0) return VX_OK;
  const int merge = p.nsplit > 1 ? units * HB : 0, chunks = (max_len + 255) / 256;
  const int blocks = merge + (track ? a.B * a.nkv * chunks : 0);
  count_launch();
  if (c->head_dim == 128)
    kv4_finish_kernel<128><<<blocks, 256, 0, st>>>(a, merge, chunks);
  else
    kv4_finish_kernel<64><<<blocks, 256, 0, st>>>(a, merge, chunks);
  VX_CUDA(ctx, cudaGetLastError());
  return VX_OK;
}

}  // extern "C"
