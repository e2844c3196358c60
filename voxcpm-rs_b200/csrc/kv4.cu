// The 4-bit KV cache: rows quantised in and read back (vx_kv4_append, vx_kv4_read).
#include <cfloat>

#include "common.cuh"
#include "kv4.cuh"
#include "runtime.cuh"

namespace vx {
namespace {

// ------------------------------------------------------------------------------- append
// Four lanes hold the 16 dims of a group, a float4 each.  amax is taken over the bit patterns
// of |x| (a NaN's are above infinity's, so a NaN in the group is not lost), the scale is
// e4m3(amax / 6), and a code is found by comparing |x| with edge * scale: an edge has at most 3
// significant bits and a scale 4, so the products are exact and a tie is seen as one.
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

// Grid (runs of a sequence's rows, sequences, keys / values).  D / 4 lanes hold a row, and a
// thread takes AP_ROWS rows a run apart, whose loads are all in flight before the first is used.
constexpr int AP_ROWS = 4;

template <int D>
__global__ void __launch_bounds__(256) kv4_append_kernel(const AppendArgs a) {
  constexpr int RPB = 256 / (D / 4);  // rows that the block holds at a time
  const int b = blockIdx.y, c = threadIdx.x % (D / 4);
  const bool is_v = blockIdx.z;
  const int n = a.counts ? a.counts[b] : a.S, at = a.start[b];
  if (n < 0 || n > a.S || at < 0 || at > a.cap - n) {
    if (blockIdx.x == 0 && threadIdx.x == 0) record_error(a.err, VX_DEVICE_ERR_BOUNDS);
    return;
  }
  const int r0 = blockIdx.x * RPB * AP_ROWS + threadIdx.x / (D / 4), rows = n * a.nkv;
  if (r0 - (int)(threadIdx.x / (D / 4)) >= rows) return;
  const float* src = (is_v ? a.v : a.k) + b * a.batch_stride + c * 4;
  float4 x[AP_ROWS];
#pragma unroll
  for (int i = 0; i < AP_ROWS; ++i) {
    const int r = r0 + i * RPB, s = r / a.nkv, h = r - s * a.nkv;
    x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (r < rows) x[i] = __ldcs(reinterpret_cast<const float4*>(src + s * a.token_stride + h * D));
  }
#pragma unroll
  for (int i = 0; i < AP_ROWS; ++i) {
    const int r = r0 + i * RPB, s = r / a.nkv, h = r - s * a.nkv;
    uint32_t m = max(max(__float_as_uint(x[i].x) & 0x7fffffffu, __float_as_uint(x[i].y) & 0x7fffffffu),
                     max(__float_as_uint(x[i].z) & 0x7fffffffu, __float_as_uint(x[i].w) & 0x7fffffffu));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
    const uint32_t s8 = __nv_cvt_float_to_fp8(__uint_as_float(m) / 6.f, __NV_SATFINITE, __NV_E4M3);
    const float sc = s8 ? e4m3_to_f32(s8) : INFINITY;  // no scale: every code is 0
    const uint32_t code = e2m1_code(x[i].x, sc) | e2m1_code(x[i].y, sc) << 4 | e2m1_code(x[i].z, sc) << 8 |
                          e2m1_code(x[i].w, sc) << 12;
    if (r >= rows) continue;
    const size_t row = ((size_t)b * a.nkv + h) * a.cap + at + s;
    reinterpret_cast<uint16_t*>((is_v ? a.v_codes : a.k_codes) + row * (D / 2))[c] = (uint16_t)code;
    if ((c & 3) == 0) (is_v ? a.v_scales : a.k_scales)[row * (D / KV4_GROUP) + c / 4] = (uint8_t)s8;
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
  if (c->batch <= 0 || c->n_kv_heads <= 0 || (long long)c->batch * c->n_kv_heads > 65535)
    return fail(ctx, VX_ERR_SHAPE, "%s: batch * n_kv_heads must lie in 1..65535", what);
  if (c->capacity <= 0 || c->capacity % 32 != 0)
    return fail(ctx, VX_ERR_SHAPE, "%s: capacity must be a positive multiple of 32 (got %d)", what, c->capacity);
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
  if ((long long)S * c->n_kv_heads > (1 << 30)) return fail(ctx, VX_ERR_SHAPE, "kv4_append: more than 2^30 rows of a sequence");
  if (S < 0 || S > c->capacity) return fail(ctx, VX_ERR_SHAPE, "kv4_append: %d tokens for %d rows", S, c->capacity);
  if ((((uintptr_t)k | (uintptr_t)v) & 15) || batch_stride % 4 != 0 || token_stride % 4 != 0)
    return fail(ctx, VX_ERR_ARG, "kv4_append: k and v must be 16-byte aligned, their strides multiples of 4");
  if (S == 0) return VX_OK;
  DeviceGuard guard(ctx->device);
  AppendArgs a = {k, v, batch_stride, token_stride, c->k_codes, c->k_scales, c->v_codes, c->v_scales, c->weights,
                  c->positions, start, counts, first_position, S, c->n_kv_heads, c->capacity, ctx->dev_err};
  const int per_block = 256 / (c->head_dim / 4) * AP_ROWS;
  const dim3 grid((S * c->n_kv_heads + per_block - 1) / per_block, c->batch, 2);
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
