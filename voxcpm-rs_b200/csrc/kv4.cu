// The 4-bit KV cache: rows quantised in and read back (vx_kv4_append, vx_kv4_read).  Both are bound by
// HBM where there is much to move: 16 ragged prompts of up to 4093 tokens (2 heads of 128) are appended
// in 14 us (75 MB) and read back in 23 us (143 MB, 6.2 TB/s); a single token of 8 sequences takes a
// launch (3.8 us for both).
#include <cfloat>

#include "common.cuh"
#include "kv4.cuh"
#include "runtime.cuh"

namespace vx {
namespace {

// ------------------------------------------------------------------------------- append
// Two lanes hold the 16 dims of a group, 8 numbers each.  amax is taken over the bit patterns of
// |x| (a NaN's are above infinity's, so a NaN in the group is not lost) and the scale is
// e4m3(amax / 6).  A code is the e2m1 number nearest to x / scale.  x / scale is not computed: x
// times a reciprocal that is 2^-21 too small and one that is as much too large enclose it, and
// where both convert to the same code that is the code; where they do not (a tie, or within 2^-21
// of one) |x| is compared with edge * scale, which is exact: an edge has at most 3 significant
// bits and a scale 4.
struct AppendArgs {
  const float* k;
  const float* v;
  long long batch_stride, token_stride;
  uint8_t *k_codes, *k_scales, *v_codes, *v_scales;
  float* weights;
  int64_t* positions;
  const int *start, *counts, *first_position;
  int S, nkv, cap;
  int* err;
};

// edges between codes j and j + 1; a tie goes to the even one, so odd edges take it
__device__ __forceinline__ uint32_t e2m1_code(float x, float s) {
  const float a = fabsf(x);
  const bool b2 = a >= 1.75f * s;
  const bool b1 = a >= (b2 ? 3.5f * s : 0.75f * s);
  const float e = b2 ? (b1 ? 5.f * s : 2.5f * s) : (b1 ? 1.25f * s : 0.25f * s);
  return (b2 ? 4u : 0u) + (b1 ? 2u : 0u) + (a > e ? 1u : 0u) + ((__float_as_uint(x) >> 28) & 8u);
}

// e2m1 codes of four numbers, the first in the lowest bits
__device__ __forceinline__ uint32_t e2m1x4(float a, float b, float c, float d) {
  uint32_t r;
  asm("{\n\t.reg .b8 lo, hi;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 lo, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 hi, %4, %3;\n\t"
      "mov.b32 %0, {lo, hi, lo, hi};\n\t}"
      : "=r"(r)
      : "f"(a), "f"(b), "f"(c), "f"(d));
  return r & 0xffffu;
}

// Grid (runs of a sequence's tokens, sequences, heads of keys and of values).  D / 8 lanes hold a
// row, and a thread takes AP_ROWS rows a run apart, whose loads are all in flight before the
// first is used.
constexpr int AP_ROWS = 2;

template <int D>
__global__ void __launch_bounds__(256) kv4_append_kernel(const AppendArgs a) {
  constexpr int LPR = D / 8, RPB = 256 / LPR;  // lanes of a row, rows that the block holds at a time
  const int b = blockIdx.y, h = blockIdx.z >> 1, c = threadIdx.x % LPR;
  const bool is_v = blockIdx.z & 1;
  const int n = a.counts ? a.counts[b] : a.S, at = a.start[b];
  if (n < 0 || n > a.S || at < 0 || at > a.cap - n) {
    if (blockIdx.x == 0 && threadIdx.x == 0) record_error(a.err, VX_DEVICE_ERR_BOUNDS);
    return;
  }
  if ((int)blockIdx.x * RPB * AP_ROWS >= n) return;
  const int s0 = blockIdx.x * RPB * AP_ROWS + threadIdx.x / LPR;
  const float* src = (is_v ? a.v : a.k) + b * a.batch_stride + h * D + c * 8;
  float4 x[AP_ROWS][2];
#pragma unroll
  for (int i = 0; i < AP_ROWS; ++i) {
    x[i][0] = x[i][1] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (s0 + i * RPB < n) {
      const float4* p = reinterpret_cast<const float4*>(src + (s0 + i * RPB) * a.token_stride);
      x[i][0] = __ldcs(p);
      x[i][1] = __ldcs(p + 1);
    }
  }
  const size_t row0 = ((size_t)b * a.nkv + h) * a.cap + at;
#pragma unroll
  for (int i = 0; i < AP_ROWS; ++i) {
    const float y[8] = {x[i][0].x, x[i][0].y, x[i][0].z, x[i][0].w, x[i][1].x, x[i][1].y, x[i][1].z, x[i][1].w};
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) m = max(m, __float_as_uint(y[e]) & 0x7fffffffu);
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    const uint32_t s8 = __nv_cvt_float_to_fp8(__uint_as_float(m) / 6.f, __NV_SATFINITE, __NV_E4M3);
    const float sc = e4m3_to_f32(s8), inv = s8 ? __frcp_rn(sc) : 0.f;  // no scale: every code is 0
    const float il = inv * (1.f - 0x1p-21f), ih = inv * (1.f + 0x1p-21f);
    uint32_t code = e2m1x4(y[0] * il, y[1] * il, y[2] * il, y[3] * il) |
                    e2m1x4(y[4] * il, y[5] * il, y[6] * il, y[7] * il) << 16;
    const uint32_t up = e2m1x4(y[0] * ih, y[1] * ih, y[2] * ih, y[3] * ih) |
                        e2m1x4(y[4] * ih, y[5] * ih, y[6] * ih, y[7] * ih) << 16;
    if (code != up) {
      code = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) code |= e2m1_code(y[e], sc) << (4 * e);
    }
    const int s = s0 + i * RPB;
    if (s >= n) continue;
    const size_t row = row0 + s;
    reinterpret_cast<uint32_t*>((is_v ? a.v_codes : a.k_codes) + row * (D / 2))[c] = code;
    if ((c & 1) == 0) (is_v ? a.v_scales : a.k_scales)[row * (D / KV4_GROUP) + c / 2] = (uint8_t)s8;
    if (c == 0 && !is_v) {
      if (a.weights) a.weights[row] = 0.f;
      if (a.positions) a.positions[row] = (int64_t)(a.first_position ? a.first_position[b] : at) + s;
    }
  }
}

// --------------------------------------------------------------------------------- read
struct ReadArgs {
  const uint8_t *k_codes, *k_scales, *v_codes, *v_scales;
  const int *start, *counts;
  float *k, *v;
  int n, nkv, cap;
  int* err;
};

// Grid (runs of rows, sequence and head, keys / values); a thread makes 4 numbers of each of
// RD_ROWS rows.
constexpr int RD_ROWS = 4;

template <int D>
__global__ void __launch_bounds__(256) kv4_read_kernel(const ReadArgs a) {
  constexpr int RPB = 256 / (D / 4);
  const int bg = blockIdx.y, b = bg / a.nkv, c = threadIdx.x % (D / 4);
  const bool is_v = blockIdx.z;
  int n = a.counts ? a.counts[b] : a.n, at = a.start ? a.start[b] : 0;
  if (n < 0 || n > a.n || at < 0 || at > a.cap - n) {
    if (blockIdx.x == 0 && threadIdx.x == 0) record_error(a.err, VX_DEVICE_ERR_BOUNDS);
    n = at = 0;  // zeros
  }
  const int r0 = blockIdx.x * RPB * RD_ROWS + threadIdx.x / (D / 4);
  const size_t row0 = (size_t)bg * a.cap + at;
  const uint8_t *codes = is_v ? a.v_codes : a.k_codes, *scales = is_v ? a.v_scales : a.k_scales;
  uint32_t w[RD_ROWS], s8[RD_ROWS];
#pragma unroll
  for (int i = 0; i < RD_ROWS; ++i) {
    const int r = r0 + i * RPB;
    w[i] = s8[i] = 0;
    if (r < n) {
      w[i] = reinterpret_cast<const uint16_t*>(codes + (row0 + r) * (D / 2))[c];
      s8[i] = scales[(row0 + r) * (D / KV4_GROUP) + c / 4];
    }
  }
  float4* out = reinterpret_cast<float4*>(is_v ? a.v : a.k) + (size_t)bg * a.n * (D / 4) + c;
#pragma unroll
  for (int i = 0; i < RD_ROWS; ++i) {
    const int r = r0 + i * RPB;
    const float sc = e4m3_to_f32(s8[i]);
    const uint32_t lo = e2m1x2_to_h2(w[i]), hi = e2m1x2_to_h2(w[i] >> 8);
    if (r < a.n)
      __stcs(out + (size_t)r * (D / 4), make_float4(h2_lo(lo) * sc, h2_hi(lo) * sc, h2_lo(hi) * sc, h2_hi(hi) * sc));
  }
}

}  // namespace

int kv4_check(vx_ctx* ctx, const vx_kv4* c, const char* what) {
  if (!ctx || !c || !c->k_codes || !c->k_scales || !c->v_codes || !c->v_scales) return VX_ERR_ARG;
  if (c->head_dim != 64 && c->head_dim != 128)
    return fail(ctx, VX_ERR_SHAPE, "%s: head_dim must be 64 or 128 (got %d)", what, c->head_dim);
  if (c->batch <= 0 || c->n_kv_heads <= 0 || c->n_kv_heads > 32767 || (long long)c->batch * c->n_kv_heads > 65535)
    return fail(ctx, VX_ERR_SHAPE, "%s: batch * n_kv_heads must lie in 1..65535 (at most 32767 heads)", what);
  if (c->capacity <= 0 || c->capacity % 32 != 0 || c->capacity > (1 << 30))
    return fail(ctx, VX_ERR_SHAPE, "%s: capacity must be a positive multiple of 32 up to 2^30 (got %d)", what,
                c->capacity);
  if (((uintptr_t)c->k_codes | (uintptr_t)c->k_scales | (uintptr_t)c->v_codes | (uintptr_t)c->v_scales) & 15)
    return fail(ctx, VX_ERR_ARG, "%s: cache buffers must be 16-byte aligned", what);
  return VX_OK;
}

}  // namespace vx

using namespace vx;

extern "C" {

int vx_kv4_append(vx_ctx* ctx, const vx_kv4* c, const float* k, const float* v, int64_t batch_stride,
                  int64_t token_stride, int S, const int32_t* start, const int32_t* counts,
                  const int32_t* first_position, vx_stream stream) {
  const int rc = kv4_check(ctx, c, "kv4_append");
  if (rc) return rc;
  if (!k || !v || !start) return fail(ctx, VX_ERR_ARG, "kv4_append: k, v and start are needed");
  if (S < 0 || S > c->capacity) return fail(ctx, VX_ERR_SHAPE, "kv4_append: %d tokens for %d rows", S, c->capacity);
  if ((((uintptr_t)k | (uintptr_t)v) & 15) || batch_stride % 4 != 0 || token_stride % 4 != 0)
    return fail(ctx, VX_ERR_ARG, "kv4_append: k and v must be 16-byte aligned, their strides multiples of 4");
  if (S == 0) return VX_OK;
  DeviceGuard guard(ctx->device);
  AppendArgs a = {k, v, batch_stride, token_stride, c->k_codes, c->k_scales, c->v_codes, c->v_scales, c->weights,
                  c->positions, start, counts, first_position, S, c->n_kv_heads, c->capacity, ctx->dev_err};
  const int per_block = 256 / (c->head_dim / 8) * AP_ROWS;
  const dim3 grid((S + per_block - 1) / per_block, c->batch, 2 * c->n_kv_heads);
  count_launch();
  if (c->head_dim == 128)
    kv4_append_kernel<128><<<grid, 256, 0, pick_stream(ctx, stream)>>>(a);
  else
    kv4_append_kernel<64><<<grid, 256, 0, pick_stream(ctx, stream)>>>(a);
  VX_CUDA(ctx, cudaGetLastError());
  return VX_OK;
}

int vx_kv4_read(vx_ctx* ctx, const vx_kv4* c, int n, const int32_t* start, const int32_t* counts, float* k, float* v,
                vx_stream stream) {
  const int rc = kv4_check(ctx, c, "kv4_read");
  if (rc) return rc;
  if (!k || !v || (((uintptr_t)k | (uintptr_t)v) & 15))
    return fail(ctx, VX_ERR_ARG, "kv4_read: k and v must be given and 16-byte aligned");
  if (n < 0 || n > c->capacity) return fail(ctx, VX_ERR_SHAPE, "kv4_read: %d of %d rows", n, c->capacity);
  if (n == 0) return VX_OK;
  DeviceGuard guard(ctx->device);
  ReadArgs a = {c->k_codes, c->k_scales, c->v_codes, c->v_scales, start, counts, k, v, n, c->n_kv_heads,
                c->capacity, ctx->dev_err};
  const int per_block = 256 / (c->head_dim / 4) * RD_ROWS;
  const dim3 grid((n + per_block - 1) / per_block, c->batch * c->n_kv_heads, 2);
  count_launch();
  if (c->head_dim == 128)
    kv4_read_kernel<128><<<grid, 256, 0, pick_stream(ctx, stream)>>>(a);
  else
    kv4_read_kernel<64><<<grid, 256, 0, pick_stream(ctx, stream)>>>(a);
  VX_CUDA(ctx, cudaGetLastError());
  return VX_OK;
}

}  // extern "C"
