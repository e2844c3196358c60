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
  int B, S, nkv, d, cap;
  int* err;
};

__device__ __forceinline__ uint32_t e2m1_code(float x, const float (&edge)[7]) {
  const float a = fabsf(x);
  // edges between codes j and j + 1; a tie goes to the even one, so odd edges take it
  uint32_t c = (a > edge[0]) + (a >= edge[1]) + (a > edge[2]) + (a >= edge[3]) + (a > edge[4]) + (a >= edge[5]) +
               (a > edge[6]);
  return c | ((__float_as_uint(x) >> 28) & 8u);
}

__global__ void __launch_bounds__(256) kv4_append_kernel(const AppendArgs a) {
  const int quads = a.d / 4;  // lanes of a row
  const long long total = (long long)a.B * a.S * a.nkv * quads * 2;
  for (long long i0 = blockIdx.x * 256LL; i0 < total; i0 += gridDim.x * 256LL) {
    const long long i = i0 + threadIdx.x;
    const bool in = i < total;
    long long r = (in ? i : 0) / quads;
    const int c = (int)((in ? i : 0) % quads);
    const int is_v = (int)(r & 1);
    r >>= 1;
    const int h = (int)(r % a.nkv);
    r /= a.nkv;
    const int s = (int)(r % a.S), b = (int)(r / a.S);
    const int n = a.counts ? a.counts[b] : a.S, at = a.start[b];
    const bool bad = n < 0 || n > a.S || at < 0 || at > a.cap - n;
    const bool live = in && !bad && s < n;
    if (in && bad && s == 0 && c == 0) record_error(a.err, VX_DEVICE_ERR_BOUNDS);
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if (live)
      x = __ldcs(reinterpret_cast<const float4*>((is_v ? a.v : a.k) + b * a.batch_stride + s * a.token_stride +
                                                 (long long)h * a.d) + c);
    uint32_t m = max(max(__float_as_uint(x.x) & 0x7fffffffu, __float_as_uint(x.y) & 0x7fffffffu),
                     max(__float_as_uint(x.z) & 0x7fffffffu, __float_as_uint(x.w) & 0x7fffffffu));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
    if (!live) continue;
    const uint32_t s8 = __nv_cvt_float_to_fp8(__uint_as_float(m) / 6.f, __NV_SATFINITE, __NV_E4M3);
    const float sc = s8 ? e4m3_to_f32(s8) : INFINITY;  // no scale: every code is 0
    const float edge[7] = {0.25f * sc, 0.75f * sc, 1.25f * sc, 1.75f * sc, 2.5f * sc, 3.5f * sc, 5.f * sc};
    const uint32_t code = e2m1_code(x.x, edge) | e2m1_code(x.y, edge) << 4 | e2m1_code(x.z, edge) << 8 |
                          e2m1_code(x.w, edge) << 12;
    const size_t row = ((size_t)b * a.nkv + h) * a.cap + at + s;
    reinterpret_cast<uint16_t*>((is_v ? a.v_codes : a.k_codes) + row * (a.d / 2))[c] = (uint16_t)code;
    if ((c & 3) == 0) (is_v ? a.v_scales : a.k_scales)[row * (a.d / KV4_GROUP) + c / 4] = (uint8_t)s8;
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
  int B, n, nkv, d, cap;
  int* err;
};

__global__ void __launch_bounds__(256) kv4_read_kernel(const ReadArgs a) {
  const int quads = a.d / 4;
  const long long half = (long long)a.B * a.nkv * a.n * quads, total = 2 * half;
  for (long long i = blockIdx.x * 256LL + threadIdx.x; i < total; i += gridDim.x * 256LL) {
    const bool is_v = i >= half;
    const long long j = is_v ? i - half : i;
    const int c = (int)(j % quads);
    long long r = j / quads;
    const int s = (int)(r % a.n);
    r /= a.n;  // b * nkv + h
    const int b = (int)(r / a.nkv);
    const int n = a.counts ? a.counts[b] : a.n, at = a.start ? a.start[b] : 0;
    const bool bad = n < 0 || n > a.n || at < 0 || at > a.cap - n;
    if (bad && s == 0 && c == 0) record_error(a.err, VX_DEVICE_ERR_BOUNDS);
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
    if (!bad && s < n) {
      const size_t row = (size_t)r * a.cap + at + s;
      const uint32_t w = reinterpret_cast<const uint16_t*>((is_v ? a.v_codes : a.k_codes) + row * (a.d / 2))[c];
      const float sc = e4m3_to_f32((is_v ? a.v_scales : a.k_scales)[row * (a.d / KV4_GROUP) + c / 4]);
      const uint32_t lo = e2m1x2_to_h2(w), hi = e2m1x2_to_h2(w >> 8);
      y = make_float4(h2_lo(lo) * sc, h2_hi(lo) * sc, h2_lo(hi) * sc, h2_hi(hi) * sc);
    }
    __stcs(reinterpret_cast<float4*>((is_v ? a.v : a.k)) + j, y);
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
  if (S < 0 || S > c->capacity) return fail(ctx, VX_ERR_SHAPE, "kv4_append: %d tokens for %d rows", S, c->capacity);
  if ((((uintptr_t)k | (uintptr_t)v) & 15) || batch_stride % 4 != 0 || token_stride % 4 != 0)
    return fail(ctx, VX_ERR_ARG, "kv4_append: k and v must be 16-byte aligned, their strides multiples of 4");
  if (S == 0) return VX_OK;
  DeviceGuard guard(ctx->device);
  AppendArgs a = {k, v, batch_stride, token_stride, c->k_codes, c->k_scales, c->v_codes, c->v_scales, c->weights,
                  c->positions, start, counts, first_position, c->batch, S, c->n_kv_heads, c->head_dim, c->capacity,
                  ctx->dev_err};
  const long long total = (long long)c->batch * S * c->n_kv_heads * (c->head_dim / 4) * 2;
  const int grid = (int)std::min<long long>((total + 255) / 256, 148 * 16);
  count_launch();
  kv4_append_kernel<<<grid, 256, 0, pick_stream(ctx, stream)>>>(a);
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
  ReadArgs a = {c->k_codes, c->k_scales, c->v_codes, c->v_scales, start, counts, k, v, c->batch, n, c->n_kv_heads,
                c->head_dim, c->capacity, ctx->dev_err};
  const long long total = (long long)c->batch * n * c->n_kv_heads * (c->head_dim / 4) * 2;
  const int grid = (int)std::min<long long>((total + 255) / 256, 148 * 32);
  count_launch();
  kv4_read_kernel<<<grid, 256, 0, pick_stream(ctx, stream)>>>(a);
  VX_CUDA(ctx, cudaGetLastError());
  return VX_OK;
}

}  // extern "C"
