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

// ------------------------------------------------------------------------------ the split
// Each warp walks its own tiles of 32 positions, with no barrier between the warps of a block
// until the end.  Both products run on m16n8k16 f16 tensor instructions with f32 sums, and are
// exact in what they multiply: a cached value has at most 6 significant bits and is made as f16
// from its code and scale; a query and a probability are split into two f16 terms (22 bits),
// and the 16 rows of an instruction are the first terms of 8 query heads and their second terms,
// whose sums are added afterwards.
//   S = Q K^T: the contracted index may be taken in any order, so thread (g, t) of the B operand
//     reads D / 4 dims of row g in one piece (16 or 8 bytes): k-step s takes its bytes 2s, 2s + 1.
//   O = P V: n-tile j's column g is dim g D/8 + j, so thread (g, t) reads one piece of 8 or 4 bytes
//     of each of its 4 positions; the pairs along positions that the operand needs are made by
//     merging the nibbles of two rows before they are converted.
//   A slot (n-tile i, column 2t + e) of S is position 8i + (e ? 7 - t : t) of a 16-position block:
//     with it both kinds of shared-memory reads are free of bank conflicts.
constexpr int AT_WARPS = 4;
constexpr int AT_TILE = 32;   // positions of a tile
constexpr int AT_STAGES = 4;  // tiles of a warp in shared memory

template <int D>
struct TileBytes {
  static constexpr int codes = AT_TILE * D / 2, scales = AT_TILE * D / 16, all = 2 * (codes + scales);
};

__device__ __forceinline__ void cp_async16(void* dst, const void* src, int bytes) {  // the rest of 16 B becomes 0
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                          uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 16-byte piece c of row r: at 64-byte rows the odd pairs of rows have their halves swapped
template <int D>
__device__ __forceinline__ int code_at(int r, int byte) {
  return D == 128 ? r * 64 + (byte ^ ((r & 2) << 4)) : r * 32 + byte;
}

// Rows [p0, p0 + 32) of one KV head into a stage; rows from p1 on are not read, their scales are 0.
template <int D>
__device__ __forceinline__ void load_tile(const AttendArgs& a, size_t row0, int p0, int p1, uint8_t* st, int lane) {
  constexpr int CPR = D / 32, SPR = D / 16;  // 16-byte pieces of a row's codes, bytes of its scales
  const size_t row = row0 + p0;
  const int nv = p1 - p0;
#pragma unroll
  for (int e = 0; e < CPR; ++e) {
    const int i = lane + 32 * e, r = i / CPR, c = i % CPR;
    const int bytes = r < nv ? 16 : 0;
    const size_t off = r < nv ? (row + r) * (D / 2) + c * 16 : row * (D / 2);
    cp_async16(st + code_at<D>(r, c * 16), a.k_codes + off, bytes);
    cp_async16(st + TileBytes<D>::codes + code_at<D>(r, c * 16), a.v_codes + off, bytes);
  }
  constexpr int SL = TileBytes<D>::scales / 16;  // lanes that bring the scales of K, and as many those of V
  if (lane < 2 * SL) {
    const int i = lane % SL;
    const int bytes = min(16, max(0, nv * SPR - i * 16));
    const uint8_t* src = (lane < SL ? a.k_scales : a.v_scales) + row * SPR + (bytes ? i * 16 : 0);
    cp_async16(st + 2 * TileBytes<D>::codes + lane * 16, src, bytes);
  }
}

template <int D>
__global__ void __launch_bounds__(AT_WARPS * 32, D == 128 ? 3 : 4) kv4_split_kernel(const AttendArgs a) {
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr int KS = D / 16, NT = D / 8;  // k-steps of S, n-tiles of O
  constexpr int OS = D + 8;               // floats of a head's row in the merge
  pdl_launch_dependents();
  const int unit = blockIdx.y, split = blockIdx.x;
  const int hb = unit % a.nhb, g0 = (unit / a.nhb) % a.nkv, b = unit / (a.nhb * a.nkv);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int n = seq_len(a, b);
  const int heads = min(HB, a.nrep - hb * HB);
  float* out = a.out + (size_t)b * a.ldo + (size_t)(g0 * a.nrep + hb * HB) * D;
  if (n <= 0) {
    if (n < 0 && tid == 0) record_error(a.err, VX_DEVICE_ERR_BOUNDS);
    if (split == 0)
      for (int i = tid; i < heads * D; i += AT_WARPS * 32) out[i] = n < 0 ? NAN : 0.f;
    return;
  }
  const int j0 = split * a.chunk, j1 = min(n, j0 + a.chunk);
  if (j0 >= j1) return;
  const size_t row0 = (size_t)(b * a.nkv + g0) * a.cap;
  uint8_t* ring = smem + warp * (AT_STAGES * TileBytes<D>::all);
  const int first = j0 + warp * AT_TILE;
  const int tiles = first < j1 ? (j1 - first + AT_WARPS * AT_TILE - 1) / (AT_WARPS * AT_TILE) : 0;
#pragma unroll
  for (int i = 0; i < AT_STAGES - 1; ++i) {
    if (i < tiles) load_tile<D>(a, row0, first + i * AT_WARPS * AT_TILE, j1, ring + i * TileBytes<D>::all, lane);
    cp_async_commit();
  }

  // the query head of this thread's rows: q times a power of two that brings its largest number to
  // 2^9 .. 2^10, in two f16 terms
  uint32_t qh[KS][2], ql[KS][2];
  float mult;  // a sum of products times this is a base-2 score
  {
    float4 q[KS];
    float amax = 0.f;
    const float* qp = a.q + (size_t)b * a.ldq + (size_t)(g0 * a.nrep + hb * HB + g) * D + t * (D / 4);
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      q[s] = g < heads ? __ldg(reinterpret_cast<const float4*>(qp) + s) : make_float4(0.f, 0.f, 0.f, 0.f);
      amax = fmaxf(amax, fmaxf(fmaxf(fabsf(q[s].x), fabsf(q[s].y)), fmaxf(fabsf(q[s].z), fabsf(q[s].w))));
    }
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    const int e = (int)(__float_as_uint(amax) >> 23);  // 255: infinity, which gives NaN below
    const int up = e == 0 ? 126 : e == 255 ? 0 : max(-126, min(126, 127 + 9 - e));
    const float f = __uint_as_float((uint32_t)(127 + up) << 23);
    mult = a.scale * __uint_as_float((uint32_t)(127 - up) << 23);
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const float v[4] = {q[s].x * f, q[s].y * f, q[s].z * f, q[s].w * f};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        qh[s][h] = pack_h2(v[2 * h], v[2 * h + 1]);
        ql[s][h] = pack_h2(v[2 * h] - h2_lo(qh[s][h]), v[2 * h + 1] - h2_hi(qh[s][h]));
      }
    }
  }

  float o[NT][4];
#pragma unroll
  for (int j = 0; j < NT; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
  float m = -INFINITY, l = 0.f;
  // this lane's row of a 16-position block in S (columns of n-tile 0; + 8 of n-tile 1), its first in O
  const int krow = (g & 1) ? 7 - (g >> 1) : (g >> 1);

  for (int it = 0; it < tiles; ++it) {
    cp_async_wait<AT_STAGES - 2>();
    __syncwarp();
    const int p0 = first + it * AT_WARPS * AT_TILE;
    const uint8_t* st = ring + (it % AT_STAGES) * TileBytes<D>::all;
    const uint8_t *kc = st, *vc = st + TileBytes<D>::codes, *ks = st + 2 * TileBytes<D>::codes,
                  *vs = ks + TileBytes<D>::scales;
    float s[8];  // n-tile i's columns 2t, 2t + 1 at 2i, 2i + 1
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 8 * i + krow;
      uint32_t w[KS / 2], sc[2];
      if constexpr (D == 128) {
        const uint4 v = *reinterpret_cast<const uint4*>(kc + code_at<D>(r, t * 16));
        w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
        const uint32_t h = e4m3x2_to_h2(*reinterpret_cast<const uint16_t*>(ks + r * 8 + 2 * t));
        sc[0] = __byte_perm(h, h, 0x1010);
        sc[1] = __byte_perm(h, h, 0x3232);
      } else {
        const uint2 v = *reinterpret_cast<const uint2*>(kc + code_at<D>(r, t * 8));
        w[0] = v.x, w[1] = v.y;
        const uint32_t one = ks[r * 4 + t];
        sc[0] = sc[1] = e4m3x2_to_h2(one | one << 8);
      }
      float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int q = 0; q < KS / 2; ++q) {
        uint32_t x[4];
        e2m1x8_to_h2(w[q], x);
        const uint32_t f = sc[q * 4 / KS];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int k = 2 * q + h;
          mma_16816(c, qh[k][0], ql[k][0], qh[k][1], ql[k][1], mul_h2(x[2 * h], f), mul_h2(x[2 * h + 1], f));
        }
      }
      s[2 * i] = (c[0] + c[2]) * mult;
      s[2 * i + 1] = (c[1] + c[3]) * mult;
    }
    if (p0 + AT_TILE > j1) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (p0 + 8 * (i >> 1) + ((i & 1) ? 7 - t : t) >= j1) s[i] = -INFINITY;
    }
    if (a.scores) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int p = p0 + 8 * (i >> 1) + ((i & 1) ? 7 - t : t);
        if (p < j1) a.scores[((size_t)unit * a.max_len + p) * HB + g] = s[i];
      }
    }
    float mt = s[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) mt = fmaxf(mt, s[i]);
    mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 1));
    mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 2));
    // the sums are rescaled only where a score has outgrown the reference by 2^8: a probability is
    // then at most 2^8, well inside f16
    if (__any_sync(0xffffffffu, mt > m + 8.f)) {
      const float mn = fmaxf(m, mt), alpha = ex2(m - mn);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[j][e] *= alpha;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      s[i] = ex2(s[i] - m);
      l += s[i];
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {  // 16 positions
      uint32_t ph[2], pl[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float x = s[4 * k + 2 * i], y = s[4 * k + 2 * i + 1];
        ph[i] = pack_h2(x, y);
        pl[i] = pack_h2(x - h2_lo(ph[i]), y - h2_hi(ph[i]));
      }
      constexpr int NW = D / 64;  // words of a thread's piece of a row
      uint32_t w[4][NW], sc[2];
#pragma unroll
      for (int e = 0; e < 4; ++e) {  // n-tile e / 2, column 2t + e % 2
        const int r = 16 * k + 8 * (e >> 1) + ((e & 1) ? 7 - t : t);
        if constexpr (D == 128) {
          const uint2 v = *reinterpret_cast<const uint2*>(vc + code_at<D>(r, g * 8));
          w[e][0] = v.x, w[e][NW - 1] = v.y;
        } else {
          w[e][0] = *reinterpret_cast<const uint32_t*>(vc + code_at<D>(r, g * 4));
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r0 = 16 * k + 8 * i + t, r1 = 16 * k + 8 * i + 7 - t;
        const uint32_t s0 = D == 128 ? vs[r0 * 8 + g] : vs[r0 * 4 + (g >> 1)];
        const uint32_t s1 = D == 128 ? vs[r1 * 8 + g] : vs[r1 * 4 + (g >> 1)];
        sc[i] = e4m3x2_to_h2(s0 | s1 << 8);
      }
#pragma unroll
      for (int q = 0; q < NW; ++q) {
        uint32_t ev[2][4], od[2][4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t x = w[2 * i][q], y = w[2 * i + 1][q];
          e2m1x8_to_h2((x & 0x0f0f0f0fu) | ((y << 4) & 0xf0f0f0f0u), ev[i]);
          e2m1x8_to_h2(((x >> 4) & 0x0f0f0f0fu) | (y & 0xf0f0f0f0u), od[i]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          mma_16816(o[8 * q + 2 * j], ph[0], pl[0], ph[1], pl[1], mul_h2(ev[0][j], sc[0]), mul_h2(ev[1][j], sc[1]));
          mma_16816(o[8 * q + 2 * j + 1], ph[0], pl[0], ph[1], pl[1], mul_h2(od[0][j], sc[0]), mul_h2(od[1][j], sc[1]));
        }
      }
    }
    __syncwarp();  // every lane has read the stage that the next load goes into
    const int nx = it + AT_STAGES - 1;
    if (nx < tiles)
      load_tile<D>(a, row0, first + nx * AT_WARPS * AT_TILE, j1, ring + (nx % AT_STAGES) * TileBytes<D>::all, lane);
    cp_async_commit();
  }
  cp_async_wait<0>();
  l += __shfl_xor_sync(0xffffffffu, l, 1);
  l += __shfl_xor_sync(0xffffffffu, l, 2);
  __syncthreads();  // the rings are free

  // merge the warps: column c = 8j + column of n-tile j of a head's row is dim (c % 8) D/8 + c / 8
  float* so = reinterpret_cast<float*>(smem);          // [warps][8][OS]
  float* sml = so + AT_WARPS * HB * OS;                 // [warps][8][2]
#pragma unroll
  for (int j = 0; j < NT; ++j)
    *reinterpret_cast<float2*>(so + (warp * HB + g) * OS + j * 8 + 2 * t) =
        make_float2(o[j][0] + o[j][2], o[j][1] + o[j][3]);
  if (t == 0) {
    sml[(warp * HB + g) * 2] = m;
    sml[(warp * HB + g) * 2 + 1] = l;
  }
  __syncthreads();
  for (int i = tid; i < heads * D; i += AT_WARPS * 32) {
    const int h = i / D, c = i % D;
    float M = -INFINITY, L = 0.f, x = 0.f;
#pragma unroll
    for (int w = 0; w < AT_WARPS; ++w) M = fmaxf(M, sml[(w * HB + h) * 2]);
#pragma unroll
    for (int w = 0; w < AT_WARPS; ++w) {
      const float f = ex2(sml[(w * HB + h) * 2] - M);
      L = fmaf(f, sml[(w * HB + h) * 2 + 1], L);
      x = fmaf(f, so[(w * HB + h) * OS + c], x);
    }
    if (a.nsplit == 1)
      out[h * D + (c % 8) * (D / 8) + c / 8] = x / L;
    else
      a.part_o[(((size_t)unit * a.nsplit + split) * HB + h) * D + c] = x;
    if (c == 0 && a.part_ml) {
      float* p = a.part_ml + (((size_t)unit * a.nsplit + split) * HB + h) * 2;
      p[0] = M;
      p[1] = L;
    }
  }
}

// Maximum and 1 / sum of one head over the active splits, by one warp.
__device__ __forceinline__ void head_stats(const AttendArgs& a, int unit, int r, int active, float* M, float* inv) {
  const int lane = threadIdx.x & 31;
  const float* p = a.part_ml + ((size_t)unit * a.nsplit * HB + r) * 2;
  float m = -INFINITY, l = 0.f;
  for (int s = lane; s < active; s += 32) m = fmaxf(m, p[(size_t)s * HB * 2]);
  m = warp_max(m);
  for (int s = lane; s < active; s += 32) l += p[(size_t)s * HB * 2 + 1] * ex2(p[(size_t)s * HB * 2] - m);
  *M = m;
  *inv = 1.f / warp_sum(l);
}

// Blocks 0 .. units * 8 - 1 merge one head each (where there is more than one split); the blocks
// behind them add the probabilities of 256 positions of one KV head to its weights.
template <int D>
__global__ void __launch_bounds__(256) kv4_finish_kernel(const AttendArgs a, int merge_blocks, int chunks) {
  __shared__ float sm[HB * 2];
  pdl_wait();
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
      const float f = ex2(a.part_ml[(((size_t)unit * a.nsplit + s) * HB + r) * 2] - M);
      const float* po = a.part_o + (((size_t)unit * a.nsplit + s) * HB + r) * D + lane * DPL;
      for (int e = 0; e < DPL; ++e) o[e] = fmaf(f, po[e], o[e]);
    }
    for (int e = 0; e < DPL; ++e) acc[warp][lane * DPL + e] = o[e];
    __syncthreads();
    if ((int)threadIdx.x < D) {
      float t = 0.f;
      for (int w = 0; w < 8; ++w) t += acc[w][threadIdx.x];
      const int c = threadIdx.x;  // the splits' columns are in the order of their n-tiles
      a.out[(size_t)b * a.ldo + (size_t)(g * a.nrep + hb * HB + r) * D + (c % 8) * (D / 8) + c / 8] = t * inv;
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
      for (int r = 0; r < heads; ++r) w += ex2(s[r] - sm[r * 2]) * sm[r * 2 + 1];
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
  // about eight rounds of three blocks per SM, a tile of each warp at least
  constexpr long long kLeast = AT_WARPS * AT_TILE;
  long long chunk = (units * max_len + 148 * 24 - 1) / (148 * 24);
  chunk = std::min<long long>(2048, (chunk + kLeast - 1) / kLeast * kLeast);
  chunk = std::max(chunk, kLeast);
  p.chunk = (int)chunk;
  p.nsplit = std::max(1, (int)((max_len + chunk - 1) / chunk));
  const bool parts = p.nsplit > 1 || track;
  p.ml_bytes = parts ? (size_t)units * p.nsplit * HB * 2 * 4 : 0;
  p.o_bytes = p.nsplit > 1 ? (size_t)units * p.nsplit * HB * c->head_dim * 4 : 0;
  p.score_bytes = track ? (size_t)units * max_len * HB * 4 : 0;
  return p;
}

}  // namespace

cudaError_t kv4_attend_configure() {
  const cudaError_t e = cudaFuncSetAttribute(kv4_split_kernel<128>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             AT_WARPS * AT_STAGES * TileBytes<128>::all);
  if (e != cudaSuccess) return e;
  return cudaFuncSetAttribute(kv4_split_kernel<64>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              AT_WARPS * AT_STAGES * TileBytes<64>::all);
}

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
  if (units > 65535) return fail(ctx, VX_ERR_SHAPE, "kv4_attend: more than 65535 blocks of 8 query heads");
  count_launch();
  if (c->head_dim == 128)
    kv4_split_kernel<128><<<dim3(p.nsplit, units), AT_WARPS * 32, AT_WARPS * AT_STAGES * TileBytes<128>::all, st>>>(a);
  else
    kv4_split_kernel<64><<<dim3(p.nsplit, units), AT_WARPS * 32, AT_WARPS * AT_STAGES * TileBytes<64>::all, st>>>(a);
  VX_CUDA(ctx, cudaGetLastError());
  if (!need || max_len == 0) return VX_OK;
  const int merge = p.nsplit > 1 ? units * HB : 0, chunks = (max_len + 255) / 256;
  PdlLaunch pl(dim3(merge + (track ? a.B * a.nkv * chunks : 0)), dim3(256), 0, st);
  count_launch();
  VX_CUDA(ctx, c->head_dim == 128 ? cudaLaunchKernelEx(&pl.cfg, kv4_finish_kernel<128>, a, merge, chunks)
                                  : cudaLaunchKernelEx(&pl.cfg, kv4_finish_kernel<64>, a, merge, chunks));
  return VX_OK;
}

}  // extern "C"
