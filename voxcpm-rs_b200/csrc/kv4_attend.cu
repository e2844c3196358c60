// Decode attention over the 4-bit KV cache (vx_kv4_attend): one query token of each sequence
// against its cached rows, s_j = scale * q . k_j, p = softmax(s), out = sum_j p_j v_j, and with
// `track` the running weight of a row += the sum of p_j over the query heads that share it.
//
// kv4_split_kernel: grid (splits, B * nkv * head blocks of up to 8 query heads); a split covers
// a run of positions.  Up to 8 splits are one thread-block cluster, which joins their (m, l, o)
// through distributed shared memory and has its scores there for `track`: one launch, no
// workspace.  More splits leave them in the workspace, and kv4_finish_kernel joins them and turns
// the scores that a tracking call left there into weights.
//
// What bounds it.  A position costs 144 bytes (d = 128) and 4 * 8 * 128 flops for 8 query heads, so HBM
// is the floor; but the products need every value as f16, twice (a query and a probability have two
// terms), and an SM does that for 16 positions in about 165 clocks, where HBM would allow 100: 32
// tensor instructions (64 clocks alone), 64 conversions and 64 multiplications by scales, which share
// the issue slots and, measured with nothing else around them, take 103 clocks together.  Long
// batches run at 3.9 TB/s (64 sequences of 32768 rows: 153 us; floor 94); short ones are bound by
// latency: launch, first tile, merge (one sequence of 64 rows 4.5 us, of 1001 rows in a cluster of
// 8 splits 5.3 us).
#include <cooperative_groups.h>

#include <cfloat>

#include "common.cuh"
#include "kv4.cuh"
#include "runtime.cuh"

namespace cg = cooperative_groups;

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
// from its code and scale; a query and a probability are split into two f16 terms (22 bits).
//   S = Q K^T: the 16 rows are the first terms of 8 query heads and their second terms, the 8
//     columns positions; the two halves are added afterwards.  The contracted index may be taken
//     in any order, so thread (g, t) of the second operand reads D / 4 dims of one row in one
//     piece (16 or 8 bytes): k-step s takes its bytes 2s, 2s + 1.
//   O^T = V^T P^T: the rows are 16 dims, the columns 8 query heads, so what S left in a thread
//     (head g, two positions of each n-tile) is its piece of the second operand, and the products
//     of both terms of P go into the same sums (a form with P as the first operand needs twice
//     the registers for them).  Thread (g, t) reads one piece of 8 or 4 bytes of each of its 4
//     positions, dims g D/8 ..; the pairs along positions that the operand needs are made by
//     merging the nibbles of two rows before they are converted.
//   Column 2t + e of n-tile i of S is position 8i + (e ? 7 - t : t) of a 16-position block: with
//     it both kinds of shared-memory reads are free of bank conflicts.
constexpr int AT_WARPS = 4;
constexpr int AT_TILE = 32;   // positions of a tile
// Tiles of a warp in shared memory.  2 where the scores of a tracking call lie beside them and all its
// blocks are on the GPU at once if four fit on an SM, not three (64 units of 4000 rows in 512 blocks: 3
// tiles 29.8 us, 2 21.8; 2 units in 16 blocks: 11.0 and 11.7; 200 ragged units in 800: 31.3 and 34.1).
constexpr int AT_STAGES = 3, AT_FEW_STAGES = 2;
constexpr int AT_MAX_CLUSTER = 8;  // splits that a cluster joins

// The dim of column c of a split's sums: columns are ordered by m-tile, then g, then the pair.
template <int D>
__device__ __forceinline__ int dim_of(int c) {
  return (c >> 1 & 7) * (D / 8) + 2 * (c >> 4) + (c & 1);
}

template <int D>
struct TileBytes {
  static constexpr int codes = AT_TILE * D / 2, scales = AT_TILE * D / 16, all = 2 * (codes + scales);
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// `bytes` of 16, the rest becomes 0
__device__ __forceinline__ void cp_async16_part(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void mma_16816_zero(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1) {  // c = A B
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
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

// Brings tiles of one KV head into a warp's stages.  A tile is one run of each of the four
// buffers, so a lane's pieces lie at fixed distances from its pointers.  Only the last tile of a
// split can be short: its rows from `nv` on are not read and their scales become 0.
template <int D>
struct TileLoader {
  static constexpr int CPL = AT_TILE * D / 2 / 512;  // 16-byte pieces of a lane: 4 or 2, of 512 bytes each
  static constexpr int SL = TileBytes<D>::scales / 16;  // lanes that bring the scales of K, and as many those of V
  const uint8_t *k, *v, *s;
  uint32_t c_dst, s_dst;
  int lane;

  __device__ __forceinline__ void init(const AttendArgs& a, size_t row, uint8_t* ring, int lane_) {
    lane = lane_;
    k = a.k_codes + row * (D / 2) + lane * 16;
    v = a.v_codes + row * (D / 2) + lane * 16;
    s = (lane < SL ? a.k_scales : a.v_scales) + row * (D / 16) + (lane % SL) * 16;
    c_dst = smem_u32(ring) + code_at<D>(lane * 16 / (D / 2), lane * 16 % (D / 2));
    s_dst = smem_u32(ring) + 2 * TileBytes<D>::codes + lane * 16;
  }
  __device__ __forceinline__ void load(int stage, int nv) {
    const uint32_t off = stage * TileBytes<D>::all;
    if (nv >= AT_TILE) {
#pragma unroll
      for (int e = 0; e < CPL; ++e) {
        cp_async16(c_dst + off + e * 512, k + e * 512);
        cp_async16(c_dst + off + TileBytes<D>::codes + e * 512, v + e * 512);
      }
      if (lane < 2 * SL) cp_async16(s_dst + off, s);
    } else {
#pragma unroll
      for (int e = 0; e < CPL; ++e) {
        const bool in = (lane * 16 + e * 512) / (D / 2) < nv;  // a piece lies in one row
        cp_async16_part(c_dst + off + e * 512, in ? k + e * 512 : k - lane * 16, in ? 16 : 0);
        cp_async16_part(c_dst + off + TileBytes<D>::codes + e * 512, in ? v + e * 512 : v - lane * 16, in ? 16 : 0);
      }
      if (lane < 2 * SL) {
        const int first = (lane % SL) * 16, bytes = min(16, max(0, nv * (D / 16) - first));
        cp_async16_part(s_dst + off, bytes ? s : s - first, bytes);
      }
    }
    k += AT_WARPS * TileBytes<D>::codes;
    v += AT_WARPS * TileBytes<D>::codes;
    s += AT_WARPS * TileBytes<D>::scales;
  }
};

template <int D, bool CLUSTER, int STAGES>
__global__ void __launch_bounds__(AT_WARPS * 32, D == 128 ? 4 : 5) kv4_split_kernel(const AttendArgs a) {
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr int KS = D / 16;  // k-steps of S, m-tiles of O^T
  constexpr int OS = D + 4;   // floats of a head's row in the merge
  pdl_launch_dependents();
  const int unit = blockIdx.y, split = blockIdx.x;
  const int hb = unit % a.nhb, g0 = (unit / a.nhb) % a.nkv, b = unit / (a.nhb * a.nkv);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int n = seq_len(a, b);
  const int heads = min(HB, a.nrep - hb * HB);
  float* out = a.out + (size_t)b * a.ldo + (size_t)(g0 * a.nrep + hb * HB) * D;
  float4 q[KS];  // on its way while the length is
  {
    const float* qp = a.q + (size_t)b * a.ldq + (size_t)(g0 * a.nrep + hb * HB + g) * D + t * (D / 4);
#pragma unroll
    for (int s = 0; s < KS; ++s)
      q[s] = g < heads ? __ldg(reinterpret_cast<const float4*>(qp) + s) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  if (n <= 0) {
    if (n < 0 && tid == 0) record_error(a.err, VX_DEVICE_ERR_BOUNDS);
    if (split == 0)
      for (int i = tid; i < heads * D; i += AT_WARPS * 32) out[i] = n < 0 ? NAN : 0.f;
    return;
  }
  const int j0 = split * a.chunk, j1 = min(n, j0 + a.chunk);
  if (!CLUSTER && j0 >= j1) return;
  const size_t row0 = (size_t)(b * a.nkv + g0) * a.cap;
  float* own_scores = reinterpret_cast<float*>(smem + AT_WARPS * STAGES * TileBytes<D>::all);  // [chunk][8]
  uint8_t* ring = smem + warp * (STAGES * TileBytes<D>::all);
  const int first = j0 + warp * AT_TILE;
  const int tiles = first < j1 ? (j1 - first + AT_WARPS * AT_TILE - 1) / (AT_WARPS * AT_TILE) : 0;
  TileLoader<D> loader;
  loader.init(a, row0 + first, ring, lane);
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) {
    if (i < tiles) loader.load(i, j1 - (first + i * AT_WARPS * AT_TILE));
    cp_async_commit();
  }

  // the query head of this thread's rows: q times a power of two that brings its largest number to
  // 2^9 .. 2^10, in two f16 terms
  uint32_t qh[KS][2], ql[KS][2];
  float mult;  // a sum of products times this is a base-2 score
  {
    float amax = 0.f;
#pragma unroll
    for (int s = 0; s < KS; ++s)
      amax = fmaxf(amax, fmaxf(fmaxf(fabsf(q[s].x), fabsf(q[s].y)), fmaxf(fabsf(q[s].z), fabsf(q[s].w))));
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

  // m-tile i: dims g D/8 + 2i (numbers 0, 1) and + 1 (2, 3) of query heads 2t (0, 2) and 2t + 1 (1, 3)
  float o[KS][4];
#pragma unroll
  for (int i = 0; i < KS; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float m = -INFINITY, l = 0.f;
  // byte offsets of this lane's pieces in a tile: its row of 8 positions in S, its two in O
  const int krow = (g & 1) ? 7 - (g >> 1) : (g >> 1);
  const int k_off = code_at<D>(krow, t * (D / 8)), ks_off = 2 * TileBytes<D>::codes + krow * (D / 16) + t * (D / 64);
  const int v_off[2] = {TileBytes<D>::codes + code_at<D>(t, g * (D / 16)),
                        TileBytes<D>::codes + code_at<D>(7 - t, g * (D / 16))};
  const int v_scales = 2 * TileBytes<D>::codes + TileBytes<D>::scales, v_group = g * (D / 8) / KV4_GROUP;
  const int vs_off[2] = {v_scales + t * (D / 16) + v_group, v_scales + (7 - t) * (D / 16) + v_group};

  for (int it = 0; it < tiles; ++it) {
    cp_async_wait<STAGES - 2>();
    __syncwarp();
    const int p0 = first + it * AT_WARPS * AT_TILE;
    const uint8_t* st = ring + (it % STAGES) * TileBytes<D>::all;
    float s[8];  // n-tile i's columns 2t, 2t + 1 at 2i, 2i + 1
#pragma unroll
    for (int i2 = 0; i2 < 2; ++i2) {  // two n-tiles at a time
      uint32_t w[2][KS / 2], sc[2][2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint8_t* p = st + (2 * i2 + e) * 8 * (D / 2);
        const uint8_t* ps = st + (2 * i2 + e) * 8 * (D / 16);
        if constexpr (D == 128) {
          const uint4 v = *reinterpret_cast<const uint4*>(p + k_off);
          w[e][0] = v.x, w[e][1] = v.y, w[e][2] = v.z, w[e][3] = v.w;
          const uint32_t h = e4m3x2_to_h2(*reinterpret_cast<const uint16_t*>(ps + ks_off));
          sc[e][0] = __byte_perm(h, h, 0x1010);
          sc[e][1] = __byte_perm(h, h, 0x3232);
        } else {
          const uint2 v = *reinterpret_cast<const uint2*>(p + k_off);
          w[e][0] = v.x, w[e][1] = v.y;
          const uint32_t one = ps[ks_off];
          sc[e][0] = sc[e][1] = e4m3x2_to_h2(one | one << 8);
        }
      }
      float c[2][4];
#pragma unroll
      for (int q = 0; q < KS / 2; ++q) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          uint32_t x[4];
          e2m1x8_to_h2(w[e][q], x);
          const uint32_t f = sc[e][q * 4 / KS];
          if (q == 0)
            mma_16816_zero(c[e], qh[0][0], ql[0][0], qh[0][1], ql[0][1], mul_h2(x[0], f), mul_h2(x[1], f));
          else
            mma_16816(c[e], qh[2 * q][0], ql[2 * q][0], qh[2 * q][1], ql[2 * q][1], mul_h2(x[0], f), mul_h2(x[1], f));
          mma_16816(c[e], qh[2 * q + 1][0], ql[2 * q + 1][0], qh[2 * q + 1][1], ql[2 * q + 1][1], mul_h2(x[2], f),
                    mul_h2(x[3], f));
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int i = 2 * i2 + e;
        s[2 * i] = (c[e][0] + c[e][2]) * mult;
        s[2 * i + 1] = (c[e][1] + c[e][3]) * mult;
      }
    }
    if (p0 + AT_TILE > j1) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (p0 + 8 * (i >> 1) + ((i & 1) ? 7 - t : t) >= j1) s[i] = -INFINITY;
    }
    if (CLUSTER ? a.weights != nullptr : a.scores != nullptr) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int p = p0 + 8 * (i >> 1) + ((i & 1) ? 7 - t : t);
        if (CLUSTER)
          own_scores[(p - j0) * HB + g] = s[i];
        else if (p < j1)
          a.scores[((size_t)unit * a.max_len + p) * HB + g] = s[i];
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
      const float a0 = __shfl_sync(0xffffffffu, alpha, 8 * t), a1 = __shfl_sync(0xffffffffu, alpha, 8 * t + 4);
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        o[i][0] *= a0, o[i][2] *= a0;
        o[i][1] *= a1, o[i][3] *= a1;
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      s[i] = ex2(s[i] - m);
      l += s[i];
    }
    uint32_t ph[2][2], pl[2][2], sc[2][2];  // 16-position block, n-tile of S in it
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float x = s[4 * k + 2 * i], y = s[4 * k + 2 * i + 1];
        ph[k][i] = pack_h2(x, y);
        pl[k][i] = pack_h2(x - h2_lo(ph[k][i]), y - h2_hi(ph[k][i]));
        const uint8_t* p = st + (2 * k + i) * 8 * (D / 16);
        sc[k][i] = e4m3x2_to_h2((uint32_t)p[vs_off[0]] | (uint32_t)p[vs_off[1]] << 8);
      }
    // The tile's products start from zero and join the running sums by plain additions: the tensor
    // core's own additions drop bits, always towards zero, and hundreds of them in a row were off
    // by 2e-6 of the result.
#pragma unroll
    for (int q = 0; q < D / 64; ++q) {  // words of a thread's piece of a row
      float c[4][4];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        uint32_t ev[2][4], od[2][4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {  // columns 2t and 2t + 1 of an n-tile
          const uint8_t* p = st + (2 * k + i) * 8 * (D / 2) + 4 * q;
          const uint32_t x = *reinterpret_cast<const uint32_t*>(p + v_off[0]);
          const uint32_t y = *reinterpret_cast<const uint32_t*>(p + v_off[1]);
          e2m1x8_to_h2((x & 0x0f0f0f0fu) | ((y << 4) & 0xf0f0f0f0u), ev[i]);
          e2m1x8_to_h2(((x >> 4) & 0x0f0f0f0fu) | (y & 0xf0f0f0f0u), od[i]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t a0 = mul_h2(ev[0][j], sc[k][0]), a1 = mul_h2(od[0][j], sc[k][0]),
                         a2 = mul_h2(ev[1][j], sc[k][1]), a3 = mul_h2(od[1][j], sc[k][1]);
          if (k == 0)
            mma_16816_zero(c[j], a0, a1, a2, a3, ph[0][0], ph[0][1]);
          else
            mma_16816(c[j], a0, a1, a2, a3, ph[1][0], ph[1][1]);
          mma_16816(c[j], a0, a1, a2, a3, pl[k][0], pl[k][1]);
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[4 * q + j][e] += c[j][e];
    }
    __syncwarp();  // every lane has read the stage that the next load goes into
    const int nx = it + STAGES - 1;
    if (nx < tiles) loader.load(nx % STAGES, j1 - (first + nx * AT_WARPS * AT_TILE));
    cp_async_commit();
  }
  cp_async_wait<0>();
  l += __shfl_xor_sync(0xffffffffu, l, 1);
  l += __shfl_xor_sync(0xffffffffu, l, 2);
  __syncthreads();  // the rings are free

  // merge the warps: column c of a head's row is dim_of<D>(c), the order in which threads hold them
  float* so = reinterpret_cast<float*>(smem);  // [warps][8][OS]
  float* sml = so + AT_WARPS * HB * OS;         // [warps][8][2]
#pragma unroll
  for (int i = 0; i < KS; ++i) {
    float* p = so + (warp * HB + 2 * t) * OS + i * 16 + 2 * g;
    *reinterpret_cast<float2*>(p) = make_float2(o[i][0], o[i][2]);
    *reinterpret_cast<float2*>(p + OS) = make_float2(o[i][1], o[i][3]);
  }
  if (t == 0) {
    sml[(warp * HB + g) * 2] = m;
    sml[(warp * HB + g) * 2 + 1] = l;
  }
  __syncthreads();
  float* joined = sml + AT_WARPS * HB * 2;  // [8][2]: maximum and sum of this block
  for (int i = tid; i < heads * (D / 4); i += AT_WARPS * 32) {
    const int h = i / (D / 4), c = i % (D / 4) * 4;
    float M = -INFINITY, L = 0.f;
#pragma unroll
    for (int w = 0; w < AT_WARPS; ++w) M = fmaxf(M, sml[(w * HB + h) * 2]);
    const float M0 = CLUSTER && j0 >= j1 ? 0.f : M;  // a block without positions: all zeros
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < AT_WARPS; ++w) {
      const float f = ex2(sml[(w * HB + h) * 2] - M0);
      const float4 y = *reinterpret_cast<const float4*>(so + (w * HB + h) * OS + c);
      L = fmaf(f, sml[(w * HB + h) * 2 + 1], L);
      x.x = fmaf(f, y.x, x.x);
      x.y = fmaf(f, y.y, x.y);
      x.z = fmaf(f, y.z, x.z);
      x.w = fmaf(f, y.w, x.w);
    }
    if (a.nsplit == 1) {
      *reinterpret_cast<float2*>(out + h * D + dim_of<D>(c)) = make_float2(x.x / L, x.y / L);
      *reinterpret_cast<float2*>(out + h * D + dim_of<D>(c + 2)) = make_float2(x.z / L, x.w / L);
    } else if (CLUSTER) {
      *reinterpret_cast<float4*>(so + h * OS + c) = x;  // read by this thread alone before
    } else {
      *reinterpret_cast<float4*>(a.part_o + (((size_t)unit * a.nsplit + split) * HB + h) * D + c) = x;
    }
    if (c == 0) {
      if (CLUSTER)
        *reinterpret_cast<float2*>(joined + h * 2) = make_float2(M, L);
      else if (a.part_ml)
        *reinterpret_cast<float2*>(a.part_ml + (((size_t)unit * a.nsplit + split) * HB + h) * 2) = make_float2(M, L);
    }
  }
  if constexpr (CLUSTER) {
    // join the splits: each block of the cluster takes a part of the columns
    cg::cluster_group cl = cg::this_cluster();
    const int C = a.nsplit, rank = (int)cl.block_rank();
    if (C > 1)
      cl.sync();
    else
      __syncthreads();
    float* fin = joined + HB * 2;  // [8][2]: maximum and 1 / sum over the cluster
    if (tid < heads) {  // where the weights or other blocks' sums need it
      float M = -INFINITY, L = 0.f;
      float2 ml[AT_MAX_CLUSTER];  // unconditional loads: one round trip for all blocks
#pragma unroll
      for (int r = 0; r < AT_MAX_CLUSTER; ++r)
        ml[r] = *reinterpret_cast<const float2*>(cl.map_shared_rank(joined, min(r, C - 1)) + tid * 2);
#pragma unroll
      for (int r = 0; r < AT_MAX_CLUSTER; ++r) M = fmaxf(M, ml[r].x);
#pragma unroll
      for (int r = 0; r < AT_MAX_CLUSTER; ++r)
        if (r < C) L = fmaf(ex2(ml[r].x - M), ml[r].y, L);
      fin[tid * 2] = M;
      fin[tid * 2 + 1] = 1.f / L;
    }
    __syncthreads();
    for (int i = rank * AT_WARPS * 32 + tid; C > 1 && i < heads * (D / 4); i += C * AT_WARPS * 32) {
      const int h = i / (D / 4), c = i % (D / 4) * 4;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
      for (int r = 0; r < C; ++r) {
        const float f = ex2(cl.map_shared_rank(joined, r)[h * 2] - fin[h * 2]);
        const float4 y = *reinterpret_cast<const float4*>(cl.map_shared_rank(so, r) + h * OS + c);
        x.x = fmaf(f, y.x, x.x);
        x.y = fmaf(f, y.y, x.y);
        x.z = fmaf(f, y.z, x.z);
        x.w = fmaf(f, y.w, x.w);
      }
      const float inv = fin[h * 2 + 1];
      *reinterpret_cast<float2*>(out + h * D + dim_of<D>(c)) = make_float2(x.x * inv, x.y * inv);
      *reinterpret_cast<float2*>(out + h * D + dim_of<D>(c + 2)) = make_float2(x.z * inv, x.w * inv);
    }
    if (a.weights) {  // one block of query heads alone: a row's weight is this block's to write
      for (int j = j0 + tid; j < j1; j += AT_WARPS * 32) {
        const float4* p = reinterpret_cast<const float4*>(own_scores + (j - j0) * HB);
        const float4 x = p[0], y = p[1];
        const float sc[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
        float w = 0.f;
#pragma unroll
        for (int h = 0; h < HB; ++h)
          if (h < heads) w += ex2(sc[h] - fin[h * 2]) * fin[h * 2 + 1];
        a.weights[row0 + j] += w;
      }
    }
    if (C > 1) cl.sync();  // the other blocks have read this one's sums
  }
}

// Maximum and 1 / sum of one head over the active splits, by one warp.
__device__ __forceinline__ void head_stats(const AttendArgs& a, int unit, int r, int active, float* M, float* inv) {
  const int lane = threadIdx.x & 31;
  const float2* p = reinterpret_cast<const float2*>(a.part_ml) + (size_t)unit * a.nsplit * HB + r;
  float m = -INFINITY, l = 0.f;
  constexpr int U = 8;
  for (int s = lane; s < active; s += 32 * U) {  // each lane's own running maximum, joined below
    float2 x[U];
#pragma unroll
    for (int i = 0; i < U; ++i) x[i] = s + 32 * i < active ? p[(size_t)(s + 32 * i) * HB] : make_float2(-INFINITY, 0.f);
    float mn = m;
#pragma unroll
    for (int i = 0; i < U; ++i) mn = fmaxf(mn, x[i].x);
    l *= ex2(m - mn);
#pragma unroll
    for (int i = 0; i < U; ++i) l = fmaf(x[i].y, ex2(x[i].x - mn), l);
    m = mn;
  }
  *M = warp_max(m);
  *inv = 1.f / warp_sum(l * ex2(m - *M));
}

// The first blocks merge the splits (where there is more than one).  Up to 32 of them: a warp for a
// head and a block for a unit's 8, lane s has split s's maximum and sum.  More: a block merges D /
// slices columns of a head, D / slices / 4 lanes read a split's and the block's groups of lanes take
// other splits.  The blocks behind them add the probabilities of a run of positions of one KV head
// to its weights, FIN_POS to a thread.
constexpr int FIN_POS = 4;
constexpr int FIN_FEW = 32;

template <int D>
__device__ __forceinline__ void merge_few(const AttendArgs& a, int unit) {
  constexpr int DPL = D / 32;
  const int h = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int hb = unit % a.nhb, g = (unit / a.nhb) % a.nkv, b = unit / (a.nhb * a.nkv);
  const int n = seq_len(a, b);
  pdl_wait();
  if (n <= 0 || h >= HB || hb * HB + h >= a.nrep) return;
  const int active = (n + a.chunk - 1) / a.chunk;
  float2 ml = make_float2(-INFINITY, 0.f);
  if (lane < active) ml = reinterpret_cast<const float2*>(a.part_ml)[((size_t)unit * a.nsplit + lane) * HB + h];
  const float M = warp_max(ml.x), f = lane < active ? ex2(ml.x - M) : 0.f;
  const float inv = 1.f / warp_sum(ml.y * f);
  const float* po = a.part_o + ((size_t)unit * a.nsplit * HB + h) * D + lane * DPL;
  float o[DPL] = {};
#pragma unroll 8
  for (int s = 0; s < active; ++s) {
    const float fs = __shfl_sync(0xffffffffu, f, s);
    const float2 x = *reinterpret_cast<const float2*>(po + (size_t)s * HB * D);
    o[0] = fmaf(fs, x.x, o[0]);
    o[1] = fmaf(fs, x.y, o[1]);
    if constexpr (DPL == 4) {
      const float2 y = *reinterpret_cast<const float2*>(po + (size_t)s * HB * D + 2);
      o[2] = fmaf(fs, y.x, o[2]);
      o[3] = fmaf(fs, y.y, o[3]);
    }
  }
  float* out = a.out + (size_t)b * a.ldo + (size_t)(g * a.nrep + hb * HB + h) * D;
#pragma unroll
  for (int e = 0; e < DPL; e += 2)
    *reinterpret_cast<float2*>(out + dim_of<D>(lane * DPL + e)) = make_float2(o[e] * inv, o[e + 1] * inv);
}

template <int D>
__global__ void __launch_bounds__(1024) kv4_finish_kernel(const AttendArgs a, int slices, int merge_blocks,
                                                          int chunks) {
  extern __shared__ __align__(16) float4 acc[];  // one for each thread
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // lengths and weights are not the split kernel's: they are read before it has ended
  if ((int)blockIdx.x < merge_blocks && a.nsplit <= FIN_FEW) {
    merge_few<D>(a, blockIdx.x);
    return;
  }
  if ((int)blockIdx.x < merge_blocks) {
    const int slice = blockIdx.x % slices, r = blockIdx.x / slices % HB, unit = blockIdx.x / (slices * HB);
    const int hb = unit % a.nhb, g = (unit / a.nhb) % a.nkv, b = unit / (a.nhb * a.nkv);
    const int n = seq_len(a, b);
    pdl_wait();
    if (n <= 0 || hb * HB + r >= a.nrep) return;
    const int active = (n + a.chunk - 1) / a.chunk;
    const int lps = D / 4 / slices, groups = blockDim.x / lps, grp = tid / lps, l4 = slice * lps + tid % lps;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    const float* ml = a.part_ml + ((size_t)unit * a.nsplit * HB + r) * 2;
    const float4* po = reinterpret_cast<const float4*>(a.part_o + ((size_t)unit * a.nsplit * HB + r) * D) + l4;
    constexpr int U = 4;  // splits of a thread on their way together, the first before the statistics are there
    float f[U];
    float4 x[U];
    auto load = [&](int s0) {
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int s = min(s0 + i * groups, active - 1);
        f[i] = s0 + i * groups < active ? ml[(size_t)s * HB * 2] : -INFINITY;
        x[i] = po[(size_t)s * HB * (D / 4)];
      }
    };
    load(grp);
    float M, inv;
    head_stats(a, unit, r, active, &M, &inv);
    for (int s = grp; s < active; s += U * groups) {
#pragma unroll
      for (int i = 0; i < U; ++i) {
        if (s + i * groups >= active) break;
        const float e = ex2(f[i] - M);
        o.x = fmaf(e, x[i].x, o.x);
        o.y = fmaf(e, x[i].y, o.y);
        o.z = fmaf(e, x[i].z, o.z);
        o.w = fmaf(e, x[i].w, o.w);
      }
      if (s + U * groups < active) load(s + U * groups);
    }
    acc[tid] = o;
    for (int half = groups / 2; half > 0; half /= 2) {  // the groups, two by two
      __syncthreads();
      if (grp < half) {
        const float4 x = acc[tid + half * lps];
        o.x += x.x, o.y += x.y, o.z += x.z, o.w += x.w;
        acc[tid] = o;
      }
    }
    if (grp == 0) {
      float* out = a.out + (size_t)b * a.ldo + (size_t)(g * a.nrep + hb * HB + r) * D;
      *reinterpret_cast<float2*>(out + dim_of<D>(l4 * 4)) = make_float2(o.x * inv, o.y * inv);
      *reinterpret_cast<float2*>(out + dim_of<D>(l4 * 4 + 2)) = make_float2(o.z * inv, o.w * inv);
    }
    return;
  }
  float* sm = reinterpret_cast<float*>(acc);  // [8][2]
  const int i = blockIdx.x - merge_blocks;
  const int c = i % chunks, bg = i / chunks, b = bg / a.nkv;
  const int n = seq_len(a, b), j0 = c * FIN_POS * (int)blockDim.x + tid;
  if (n <= 0 || j0 - tid >= n) {
    pdl_wait();
    return;
  }
  const int active = (n + a.chunk - 1) / a.chunk;
  float w[FIN_POS], got[FIN_POS];
#pragma unroll
  for (int u = 0; u < FIN_POS; ++u) {
    const int j = j0 + u * blockDim.x;
    w[u] = j < n ? a.weights[(size_t)bg * a.cap + j] : 0.f;
    got[u] = 0.f;
  }
  pdl_wait();
  for (int hb = 0; hb < a.nhb; ++hb) {
    const int unit = bg * a.nhb + hb, heads = min(HB, a.nrep - hb * HB);
    float4 s[FIN_POS][2];
#pragma unroll
    for (int u = 0; u < FIN_POS; ++u) {
      const int j = min(j0 + u * (int)blockDim.x, n - 1);
      const float4* p = reinterpret_cast<const float4*>(a.scores + ((size_t)unit * a.max_len + j) * HB);
      s[u][0] = p[0];
      s[u][1] = p[1];
    }
    __syncthreads();
    for (int h = warp; h < heads; h += blockDim.x / 32) {
      float M, inv;
      head_stats(a, unit, h, active, &M, &inv);
      if (lane == 0) {
        sm[h * 2] = M;
        sm[h * 2 + 1] = inv;
      }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < FIN_POS; ++u) {
      const float x[8] = {s[u][0].x, s[u][0].y, s[u][0].z, s[u][0].w, s[u][1].x, s[u][1].y, s[u][1].z, s[u][1].w};
#pragma unroll
      for (int h = 0; h < HB; ++h)
        if (h < heads) got[u] += ex2(x[h] - sm[h * 2]) * sm[h * 2 + 1];
    }
  }
#pragma unroll
  for (int u = 0; u < FIN_POS; ++u) {
    const int j = j0 + u * blockDim.x;
    if (j < n) a.weights[(size_t)bg * a.cap + j] = w[u] + got[u];
  }
}

constexpr int AT_CLUSTER_CHUNK = 512;  // their positions at most: the scores of a tracking call lie in shared memory

struct AttendPlan {
  int nhb, chunk, nsplit;
  bool cluster;
  size_t ml_bytes, o_bytes, score_bytes;
  size_t need() const { return ml_bytes + o_bytes + score_bytes; }
};

AttendPlan plan_of(const vx_kv4* c, int nh, int max_len, int track) {
  AttendPlan p = {};
  constexpr int kLeast = AT_WARPS * AT_TILE;  // a tile for each warp
  const int nrep = nh / c->n_kv_heads;
  p.nhb = (nrep + HB - 1) / HB;
  const long long units = (long long)c->batch * c->n_kv_heads * p.nhb;
  // Short sequences: the most splits, as long as all blocks are on the GPU at once, four to an SM
  // (8 sequences of 1024 rows: 8 splits in a cluster 7.0 us, through the workspace 7.1 us and one
  // launch more, 1 split of 1024 rows 10.5 us).
  auto chunk_of = [&](int splits) {
    const long long run = (long long)splits * kLeast;
    return std::max(1ll, (max_len + run - 1) / run) * kLeast;
  };
  int splits = AT_MAX_CLUSTER;
  while (splits > 1 && (units * splits > 148 * 4 || (splits / 2) * kLeast >= max_len) &&
         chunk_of(splits / 2) <= AT_CLUSTER_CHUNK)
    splits /= 2;
  // (several blocks of query heads would add to the same weights: not in a cluster)
  if (chunk_of(splits) <= AT_CLUSTER_CHUNK && p.nhb == 1) {
    p.cluster = true;
    p.chunk = (int)chunk_of(splits);
    p.nsplit = splits;
    return p;
  }
  // Long ones.  One sequence or two: the shortest splits of which two to an SM are all (1 of 131071 rows:
  // 512 positions 18.9 us, 896 16.8; of 40000: 512 11.6, 384 10.4; 8 heads of 131071: 896 48.0, 3584 45.4;
  // 2 of up to 65536: 512 19.0, 896 16.5; but 4 ragged ones of up to 32768: 512 21.0, 896 23.6).
  auto splits_of = [&](long long chunk) { return (max_len + chunk - 1) / chunk; };
  long long chunk = 0;
  if (c->batch <= 2) {
    chunk = std::max(1ll, units * max_len / (148 * 2 * kLeast)) * kLeast;
    while (chunk <= 4096 && units * splits_of(chunk) > 148 * 2) chunk += kLeast;
  }
  // More, which may differ in length: two rounds of blocks, of 512 to 4096 positions (a block costs about
  // 5 us next to its tiles; 64 sequences of 32768 rows: 512 positions 167 us, 4096 139 us; 32 ragged ones
  // of up to 8191: 512 27 us, 4096 47 us; the sums of more splits than 256 cost more to merge than they
  // save)
  if (chunk == 0 || chunk > (c->batch == 1 ? 4096 : 1024)) {
    chunk = (units * max_len + 148 * 8 - 1) / (148 * 8);
    const long long least = units * max_len <= 148 * 4 * kLeast ? kLeast : 512;
    chunk = std::min<long long>(4096, std::max(least, (chunk + kLeast - 1) / kLeast * kLeast));
  }
  p.chunk = (int)chunk;
  p.nsplit = std::max(1, (int)splits_of(chunk));
  p.ml_bytes = p.nsplit > 1 || track ? (size_t)units * p.nsplit * HB * 2 * 4 : 0;
  p.o_bytes = p.nsplit > 1 ? (size_t)units * p.nsplit * HB * c->head_dim * 4 : 0;
  p.score_bytes = track ? (size_t)units * max_len * HB * 4 : 0;
  return p;
}

constexpr size_t split_smem(int d, int stages) {
  return AT_WARPS * stages * (d == 128 ? TileBytes<128>::all : TileBytes<64>::all);
}
constexpr size_t cluster_smem(int d, int stages, int chunk, bool track) {
  return split_smem(d, stages) + (track ? (size_t)chunk * HB * 4 : 0);
}

template <int D>
cudaError_t launch_split(const AttendArgs& a, const AttendPlan& p, int units, cudaStream_t st) {
  if (!p.cluster) {
    kv4_split_kernel<D, false, AT_STAGES>
        <<<dim3(p.nsplit, units), AT_WARPS * 32, split_smem(D, AT_STAGES), st>>>(a);
    return cudaGetLastError();
  }
  const int blocks = units * p.nsplit;
  const bool track = a.weights != nullptr, few = D == 128 && track && blocks > 148 * 3 && blocks <= 148 * 4;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.nsplit, units);
  cfg.blockDim = dim3(AT_WARPS * 32);
  cfg.dynamicSmemBytes = cluster_smem(D, few ? AT_FEW_STAGES : AT_STAGES, p.chunk, track);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.nsplit;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.nsplit > 1 ? 1 : 0;
  if constexpr (D == 128)
    if (few) return cudaLaunchKernelEx(&cfg, kv4_split_kernel<D, true, AT_FEW_STAGES>, a);
  return cudaLaunchKernelEx(&cfg, kv4_split_kernel<D, true, AT_STAGES>, a);
}

template <int D>
cudaError_t configure_split() {
  const int most = (int)cluster_smem(D, AT_STAGES, AT_CLUSTER_CHUNK, true);
  auto allow = [&](void (*kernel)(AttendArgs)) {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
  };
  cudaError_t e = allow(kv4_split_kernel<D, false, AT_STAGES>);
  if (e == cudaSuccess) e = allow(kv4_split_kernel<D, true, AT_STAGES>);
  if constexpr (D == 128)
    if (e == cudaSuccess) e = allow(kv4_split_kernel<D, true, AT_FEW_STAGES>);
  return e;
}

}  // namespace

cudaError_t kv4_attend_configure() {
  const cudaError_t e = configure_split<128>();
  return e != cudaSuccess ? e : configure_split<64>();
}

}  // namespace vx

using namespace vx;

extern "C" {

size_t vx_kv4_attend_workspace(const vx_kv4* c, int nh, int max_len, int track) {
  if (!c || c->n_kv_heads <= 0 || nh <= 0 || nh % c->n_kv_heads != 0 || max_len < 0 || c->batch <= 0) return 0;
  return plan_of(c, nh, max_len, track).need();
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
      out_stride < (int64_t)nh * c->head_dim)
    return fail(ctx, VX_ERR_ARG, "kv4_attend: the rows of q and out must be 16-byte aligned, those of out not overlap");
  const AttendPlan p = plan_of(c, nh, max_len, track);
  const size_t need = p.need();
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
  VX_CUDA(ctx, c->head_dim == 128 ? launch_split<128>(a, p, units, st) : launch_split<64>(a, p, units, st));
  if (!need || max_len == 0) return VX_OK;
  // few units with many splits: more blocks to a head, and more groups of lanes in them
  const int slices = units <= 16 ? c->head_dim / 32 : 1;
  int threads = 256;
  while (p.nsplit > FIN_FEW && threads < 1024 && threads / (c->head_dim / 4 / slices) * 4 < p.nsplit) threads *= 2;
  const int merge = p.nsplit == 1 ? 0 : p.nsplit <= FIN_FEW ? units : units * HB * slices;
  const int chunks = (int)(((long long)max_len + FIN_POS * threads - 1) / (FIN_POS * threads));
  PdlLaunch pl(dim3(merge + (track ? a.B * a.nkv * chunks : 0)), dim3(threads), threads * sizeof(float4), st);
  count_launch();
  VX_CUDA(ctx, c->head_dim == 128 ? cudaLaunchKernelEx(&pl.cfg, kv4_finish_kernel<128>, a, slices, merge, chunks)
                                  : cudaLaunchKernelEx(&pl.cfg, kv4_finish_kernel<64>, a, slices, merge, chunks));
  return VX_OK;
}

}  // extern "C"
