// Token sampling from logits (vx_sample): temperature, top-k, top-p, min-p and a draw from a
// given random number, one cluster of thread blocks per row of logits.
//
// A token's weight is w = rint(exp((l - lmax) / T) * 2^44) as a 64-bit integer: sums of weights
// are exact whatever their order (a row of 2^18 tokens stays below 2^62), so every block and
// every order of atomics finds the same border.  The tokens that stay are a prefix of the order
// (logit descending, index ascending), described by the last of them, an "entry": the logit's
// ordered bits above the inverted index.
//
// The border is found by counts (top-k) or weights (top-p): a histogram of lmax - l in equal
// buckets says in which bucket it lies, and the few entries of that bucket are gathered, sorted
// and summed by one block.  Where top-k leaves few tokens these are gathered at once, and top-p,
// min-p and the draw work on the sorted list.  A bucket too full for the list (equal logits, or a
// border behind the range of the buckets) goes through radix passes over the entries instead.
// The draw takes the first token in index order whose running sum of staying weights exceeds
// u * total: sums of each warp's part of the row, then one block walks the part that holds it.
//
// What bounds it: with many rows of which every token needs its weight, instruction issue and latency in
// the pass that computes it (11 f64 operations and a table read for each token), the shared-memory
// atomics of the counting pass before, and the read, which take about 60, 50 and 37 thousand clocks of
// a block (256 rows of 151643 tokens 183 us, where reading them alone takes 24); with few rows the round
// trips between the blocks (each about half a microsecond; six of them; one row of 73448 tokens 14 us).
// A 64-bit sum takes two 32-bit atomics, 3.7 clocks of an SM for 32 tokens, where one 64-bit atomic is
// a compare-and-swap loop of 30.
#include <cooperative_groups.h>

#include <cfloat>

#include "common.cuh"
#include "runtime.cuh"

namespace cg = cooperative_groups;

namespace vx {
namespace {

typedef unsigned long long u64;

constexpr int SP_MAX_CLUSTER = 8;
constexpr int SP_MAX_VOCAB = 1 << 18;  // sums of weights stay below 2^62
constexpr int SP_THREADS = 512;
constexpr int SP_BITS = 44;          // binary places of a weight
constexpr int SP_MIDDLE_SLICE = 12288;  // tokens of a block for which another exponential each costs more than a longer list
constexpr double SP_ONE = (double)(1ull << SP_BITS);

// 2^(i / 16)
__constant__ double kExpTable[16] = {
    1.0, 1.0442737824274138, 1.0905077326652577, 1.1387886347566916, 1.189207115002721,
    1.241857812073484, 1.2968395546510096, 1.3542555469368927, 1.4142135623730951, 1.4768261459394993,
    1.5422108254079407, 1.6104903319492543, 1.681792830507429, 1.7562521603732995, 1.8340080864093424, 1.9152065613971474};

struct SampleArgs {
  const float* logits;
  long long ld;
  int rows, vocab, slice;
  const float* u;   // [rows], or with `step` a row of them for each step
  const int* step;  // device step of a decode loop, or null
  const float* temperature;
  const int* top_k;
  const float *top_p, *min_p;
  int* ids;
  float* logprob;
};

// Ascending with the logit, then descending with the index; -0 and 0 are the same.
__device__ __forceinline__ u64 entry_of(float l, int index) {
  const uint32_t u = __float_as_uint(l + 0.f), k = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return (u64)k << 24 | (0xffffffu - (uint32_t)index);
}
__device__ __forceinline__ float logit_of(u64 entry) {
  const uint32_t k = (uint32_t)(entry >> 24);
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
__device__ __forceinline__ int index_of(u64 entry) { return 0xffffff - (int)(entry & 0xffffffu); }

// Two forms.  Few rows: the row in shared memory, where three passes read it.  Many rows: read from
// L2 after the first pass, which leaves room for twice the buckets and so for a shorter list.
template <bool IN_SHARED>
struct SampleShared {
  static constexpr bool kFewRows = IN_SHARED;
  static constexpr int kThreads = SP_THREADS, kWarps = SP_THREADS / 32;
  static constexpr int kBuckets = IN_SHARED ? 2048 : 4096, kCoarse = kBuckets / 32;
  static constexpr int kList = IN_SHARED ? 1024 : 512;  // entries that are sorted
  union {
    struct {
      uint32_t lo[kBuckets], hi[kBuckets];
    } hist;
    struct {
      u64 wt[kList], pre[kList];  // of the sorted list: weights, running sums
    } list;
  };
  u64 ent[kList];  // gathered entries
  double tab[16];    // 2^(i / 16)
  float kept[kWarps][64];               // logits whose weights a warp has yet to sum
  uint32_t part_lo[kWarps], part_hi[kWarps];  // the sum of each warp's part of the row
  u64 coarse[kCoarse];
  u64 warp64[kWarps], warp_sure[kWarps];
  u64 total, above, border;
  u64 block_sum, run;  // of the draw: staying weight of this block, and before the part that holds the token
  float into;  // how far into its bucket find_bucket's border lies
  uint32_t warp32[kWarps];
  float fmax, fmin;
  int bad, bucket, n;
};

// Everything that the passes over a row share.
extern __shared__ __align__(16) float shared_row[];

template <bool IN_SHARED>
struct Row {
  const float* x;  // this block's logits
  int lo, cnt;     // their first index and number
  float lmax, floor_;
  double lmax_d, inv_t, per_16th;  // 1 / T; 16 / (T ln 2)
  const double* tab;

  __device__ __forceinline__ float at(int j) const { return IN_SHARED ? shared_row[j] : __ldg(x + j); }

  // exp(d / T) by a table of 2^(i/16) and a polynomial (table-driven, after Tang, 1989): with d / T in
  // units of ln 2 / 16 split into an integer and x in [-1/2, 1/2], 2^(x/16) = 1 + x (c1 + .. + c5 x^4),
  // Chebyshev's interpolation, off by less than 2^-46 of itself.  16 table entries of 8 bytes are all
  // banks of shared memory once: a warp reads them without conflicts (a table of 64 with fewer terms
  // took longer).  A token at z = d / T <= -31.5 has no weight (exp(-31.2) 2^44 = 1/2), nor has one
  // next to +infinity or -infinity itself, where z is infinite or a NaN.
  // floor_: where lmax and the temperature are finite and ordinary, a logit at which z is below
  // -31.5, so that none from there down has a weight; else -infinity, and the cases are told apart.
  __device__ __forceinline__ u64 weight(float l) const {
    if (floor_ > -INFINITY) return l > floor_ ? exp_of((double)l - lmax_d) : 0;
    const double d = l == lmax ? 0.0 : (double)l - lmax_d;
    return d * inv_t > -31.5 ? exp_of(d) : 0;
  }
  __device__ __forceinline__ u64 exp_of(double d) const {
    constexpr double kShift = 6755399441055744.0;  // 1.5 * 2^52: a sum with it is rounded to an integer
    const double t = fma(d, per_16th, kShift);
    const int n = __double2loint(t);
    const double x = fma(d, per_16th, kShift - t);
    double p = fma(x, 1.2716049516906705e-09, 1.4676387238435006e-07);
    p = fma(p, x, 1.3550807778387664e-05);
    p = fma(p, x, 0.0009383847926296646);
    p = fma(p, x, 0.04332169878499658);
    p = fma(p, x, 1.0);
    const double e = tab[n & 15];
    const double s = __hiloint2double(__double2hiint(e) + ((n & ~15) << 16) + (SP_BITS << 20), __double2loint(e));
    const double w = fma(p, s, 4503599627370496.0);  // + 2^52: the nearest integer, in the low bits
    return (u64)(__double2hiint(w) & 0xfffff) << 32 | (uint32_t)__double2loint(w);
  }
};

__device__ __forceinline__ u64 warp_sum64(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ u64 warp_scan64(u64 v) {  // inclusive
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 t = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += t;
  }
  return v;
}

// Adds to a 64-bit sum in two words; the word of the carry is touched where there is something to add.
__device__ __forceinline__ void add64(uint32_t* lo, uint32_t* hi, u64 v) {
  const uint32_t l = (uint32_t)v, old = atomicAdd(lo, l);
  const uint32_t h = (uint32_t)(v >> 32) + (old + l < l);
  if (h) atomicAdd(hi, h);
}

// Equal buckets of lmax - l: at `per` buckets to a unit, the last one holds the rest.
template <class Shared>
struct Buckets {
  float lmax, per;
  __device__ __forceinline__ float place(float l) const {
    return l == lmax ? 0.f : fminf((lmax - l) * per, (float)(Shared::kBuckets - 1));
  }
  __device__ __forceinline__ int operator()(float l) const { return (int)place(l); }
};

// What find_bucket adds up: tokens, their weights (PLAIN: in a row without special cases), or, in such a
// row, for each token the weight at the middle of its bucket, which needs no exponential of its own.
enum { SP_TOKENS, SP_WEIGHTS, SP_PLAIN, SP_MIDDLES };

// The histogram over the cluster of value(l, index) and the bucket in which the running sum from
// the largest logit on reaches need(total): s.bucket, s.above (the sum before it), s.total.  Every
// block finds the same.
template <int KIND, class Shared, class R, class Value, class Need>
__device__ void find_bucket(cg::cluster_group& cl, Shared& s, const R& row, const Buckets<Shared>& bucket, Value value,
                            Need need) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, C = (int)cl.num_blocks();
  for (int i = tid; i < Shared::kBuckets; i += Shared::kThreads) s.hist.lo[i] = s.hist.hi[i] = 0;
  __syncthreads();
  constexpr int U = 4;  // logits of a thread that are on their way together
  // middles: the few tokens of weight above exp(-6) are added by an f32 exponential, since a large one's
  // middle may be half a percent of all off; to 28 places, of which each word of a sum takes 14, so that
  // 2^18 of them fit and no carry is needed
  const int exact = KIND == SP_MIDDLES ? (int)fminf((float)(6.0 / row.inv_t) * bucket.per, (float)Shared::kBuckets) : 0;
  const float per_two = KIND == SP_MIDDLES ? (float)(-1.4426950408889634 * row.inv_t) : 0.f;
  constexpr bool AHEAD = KIND == SP_MIDDLES;  // read from L2: loads one round ahead
  float next[U];
  auto load = [&](int j0) {
#pragma unroll
    for (int i = 0; i < U; ++i) next[i] = j0 + i * Shared::kThreads < row.cnt ? row.at(j0 + i * Shared::kThreads) : -INFINITY;
  };
  if (AHEAD) load(tid);
  for (int j0 = tid; j0 < row.cnt; j0 += U * Shared::kThreads) {
    if (!AHEAD) load(j0);
    float l[U];
#pragma unroll
    for (int i = 0; i < U; ++i) l[i] = next[i];
    if (AHEAD) load(j0 + U * Shared::kThreads);
    // plain rows: `per` is finite and no logit above the floor lies behind the last bucket
    if constexpr (KIND == SP_MIDDLES) {
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (l[i] > row.floor_) {
          const float d = bucket.lmax - l[i];
          const int at = (int)(d * bucket.per);
          if (at >= exact) {
            atomicAdd(&s.hist.lo[at], 1u);
          } else {
            const uint32_t w = (uint32_t)exp2f(fmaf(d, per_two, 28.f));
            atomicAdd(&s.hist.lo[at], w & 0x3fff);
            atomicAdd(&s.hist.hi[at], w >> 14);
          }
        }
    } else if constexpr (KIND == SP_PLAIN) {
      u64 v[U];
#pragma unroll
      for (int i = 0; i < U; ++i) v[i] = row.exp_of((double)fmaxf(l[i], row.floor_) - row.lmax_d);
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (l[i] > row.floor_) {
          const int at = (int)((bucket.lmax - l[i]) * bucket.per);
          add64(&s.hist.lo[at], &s.hist.hi[at], v[i]);
        }
    } else {
      u64 v[U];
#pragma unroll
      for (int i = 0; i < U; ++i) v[i] = l[i] > -INFINITY ? value(l[i], row.lo + j0 + i * Shared::kThreads) : 0;
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int at = bucket(l[i]);
        if (v[i] && KIND == SP_WEIGHTS) add64(&s.hist.lo[at], &s.hist.hi[at], v[i]);
        if (v[i] && KIND == SP_TOKENS) atomicAdd(&s.hist.lo[at], (uint32_t)v[i]);
      }
    }
  }
  if constexpr (KIND == SP_MIDDLES) {
    __syncthreads();
    for (int i = tid; i < Shared::kBuckets; i += Shared::kThreads) {
      u64 v = 0;
      if (i < exact)
        v = (((u64)s.hist.hi[i] << 14) + s.hist.lo[i]) << (SP_BITS - 28);
      else if (s.hist.lo[i])
        v = s.hist.lo[i] * row.exp_of(-(i + 0.5) / bucket.per);
      s.hist.lo[i] = (uint32_t)v;
      s.hist.hi[i] = (uint32_t)(v >> 32);
    }
  }
  __syncthreads();
  for (int c = warp; c < Shared::kCoarse; c += Shared::kWarps) {
    const int i = c * (Shared::kBuckets / Shared::kCoarse) + lane;
    const u64 v = warp_sum64((u64)s.hist.hi[i] << 32 | s.hist.lo[i]);
    if (lane == 0) s.coarse[c] = v;
  }
  cl.sync();
  // Few rows: clusters of up to 8, whose blocks are all read by unconditional loads, on their way together
  // (one row 15.9 -> 14.0 us).  Many rows: clusters of 2, as a rule, so the others' loads are passed over.
  if (warp == 0) {
    constexpr int CL = Shared::kCoarse / 32;  // coarse sums of a lane
    u64 v[CL] = {}, sum = 0;
#pragma unroll
    for (int r = 0; r < SP_MAX_CLUSTER; ++r) {
      if (!Shared::kFewRows && r >= C) continue;
      const u64* p = cl.map_shared_rank(s.coarse, Shared::kFewRows ? min(r, C - 1) : r) + lane * CL;
#pragma unroll
      for (int e = 0; e < CL; ++e) v[e] += r < C ? p[e] : 0;
    }
#pragma unroll
    for (int e = 0; e < CL; ++e) sum += v[e];
    const u64 incl = warp_scan64(sum), total = __shfl_sync(0xffffffffu, incl, 31), want = need(total);
    const uint32_t hit = __ballot_sync(0xffffffffu, incl >= want);
    const int at = hit ? __ffs(hit) - 1 : 31;  // (always one: want is at most the total)
    u64 above = incl - sum;
    int c = lane * CL;
    bool past = true;
#pragma unroll
    for (int e = 0; e < CL - 1; ++e) {
      past = past && above + v[e] < want;
      if (past) above += v[e], ++c;
    }
    above = __shfl_sync(0xffffffffu, above, at);
    c = __shfl_sync(0xffffffffu, c, at);
    const int i = c * (Shared::kBuckets / Shared::kCoarse) + lane;
    u64 f = 0;
#pragma unroll
    for (int r = 0; r < SP_MAX_CLUSTER; ++r) {
      if (!Shared::kFewRows && r >= C) continue;
      const int q = Shared::kFewRows ? min(r, C - 1) : r;
      const u64 x = (u64)cl.map_shared_rank(s.hist.hi, q)[i] << 32 | cl.map_shared_rank(s.hist.lo, q)[i];
      f += r < C ? x : 0;
    }
    const u64 fi = warp_scan64(f) + above;
    const uint32_t fh = __ballot_sync(0xffffffffu, fi >= want);
    const int b = fh ? __ffs(fh) - 1 : 31;
    const u64 before = __shfl_sync(0xffffffffu, fi - f, b), own = __shfl_sync(0xffffffffu, f, b);
    if (lane == 0) {
      s.into = (float)((double)(want - before) / (double)own);
      s.bucket = c * (Shared::kBuckets / Shared::kCoarse) + b;
      s.above = before;
      s.total = total;
    }
  }
  __syncthreads();
}

// A warp's lanes for which `in` holds put their entries behind this block's others.
template <class Shared>
__device__ __forceinline__ void append(Shared& s, bool in, float l, int index) {
  const uint32_t m = __ballot_sync(0xffffffffu, in);
  if (m == 0) return;
  const int lane = threadIdx.x & 31;
  int at = 0;
  if (lane == __ffs(m) - 1) at = atomicAdd(&s.n, __popc(m));
  at = __shfl_sync(0xffffffffu, at, __ffs(m) - 1) + __popc(m & ((1u << lane) - 1));
  if (in && at < Shared::kList) s.ent[at] = entry_of(l, index);
}

// The blocks' entries, in no order, in block 0's s.ent; their number, the same for all.  Above
// Shared::kList the list is of no use.
template <class Shared>
__device__ int collect(cg::cluster_group& cl, Shared& s) {
  const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  cl.sync();
  int first[SP_MAX_CLUSTER + 1];
  first[0] = 0;
#pragma unroll
  for (int r = 0; r < SP_MAX_CLUSTER; ++r) {
    const int n = !Shared::kFewRows && r >= C ? 0 : *cl.map_shared_rank(&s.n, Shared::kFewRows ? min(r, C - 1) : r);
    first[r + 1] = r < C ? n : 0;
  }
#pragma unroll
  for (int r = 0; r < SP_MAX_CLUSTER; ++r) first[r + 1] += first[r];
  const int n = first[SP_MAX_CLUSTER];
  if (rank == 0 && n <= Shared::kList) {
    for (int i = first[1] + threadIdx.x; i < n; i += Shared::kThreads) {
      int owner = 0, at = i;
#pragma unroll
      for (int r = 1; r < SP_MAX_CLUSTER; ++r)
        if (i >= first[r]) owner = r, at = i - first[r];
      s.ent[i] = cl.map_shared_rank(s.ent, owner)[at];
    }
  }
  __syncthreads();
  return n;
}

template <class Shared, class R, class Take>
__device__ int gather(cg::cluster_group& cl, Shared& s, const R& row, Take take) {
  if (threadIdx.x == 0) s.n = 0;
  __syncthreads();
  constexpr int U = 4;
  for (int j0 = 0; j0 < row.cnt; j0 += U * Shared::kThreads) {
    float l[U];
    bool in[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int j = j0 + i * Shared::kThreads + threadIdx.x;
      l[i] = j < row.cnt ? row.at(j) : -INFINITY;
      in[i] = j < row.cnt && take(l[i], row.lo + j);
    }
#pragma unroll
    for (int i = 0; i < U; ++i) append(s, in[i], l[i], row.lo + j0 + i * Shared::kThreads + threadIdx.x);
  }
  return collect(cl, s);
}

// The sum of the weights, where at least `least`, of the logits j in [j0, j1) for which keep(l, j)
// holds, by one warp.  The few that are kept are first put side by side, 32 for each exponential.
template <class Shared, class R, class Keep>
__device__ u64 sum_kept(Shared& s, const R& row, int j0, int j1, u64 least, Keep keep) {
  const int lane = threadIdx.x & 31;
  float* buf = s.kept[threadIdx.x >> 5];
  int n = 0;
  u64 sum = 0;
  auto add = [&](bool in, float l) {
    const u64 w = in ? row.weight(l) : 0;
    if (w >= least) sum += w;
  };
  for (int j = j0 + lane; j - lane < j1; j += 32) {
    const float l = j < j1 ? row.at(j) : -INFINITY;
    const bool in = keep(l, j) && j < j1;
    const uint32_t m = __ballot_sync(0xffffffffu, in);
    if (in) buf[n + __popc(m & ((1u << lane) - 1))] = l;
    n += __popc(m);
    if (n >= 32) {
      n -= 32;
      __syncwarp();
      add(true, buf[n + lane]);
      __syncwarp();
    }
  }
  __syncwarp();
  add(lane < n, buf[lane]);
  __syncwarp();
  return warp_sum64(sum);
}

// A warp's sums over the logits j in [j0, j1) of a row without special cases, each weight computed
// once: of all, of those before bucket `from`, and of the latter the weights of at least `least`.
// Those in buckets [from, behind) go on the list.
struct Sums {
  u64 all, sure, kept;
};
template <bool MIN_P, class Shared, class R>
__device__ Sums sum_all(Shared& s, const R& row, const Buckets<Shared>& bucket, int j0, int j1, float from, float behind,
                        u64 least) {
  constexpr int U = 4;
  const int lane = threadIdx.x & 31;
  Sums t = {0, 0, 0};
  float next[U];
  auto load = [&](int j) {
#pragma unroll
    for (int i = 0; i < U; ++i) next[i] = j + 32 * i < j1 ? row.at(j + 32 * i) : -INFINITY;
  };
  load(j0 + lane);
  for (int j = j0 + lane; j - lane < j1; j += U * 32) {
    float l[U], at[U];
    u64 w[U];
#pragma unroll
    for (int i = 0; i < U; ++i) l[i] = next[i];
    load(j + U * 32);
#pragma unroll
    for (int i = 0; i < U; ++i) {
      w[i] = row.exp_of((double)fmaxf(l[i], row.floor_) - row.lmax_d);  // 0 at the floor
      at[i] = (bucket.lmax - l[i]) * bucket.per;
    }
    bool some = false;
#pragma unroll
    for (int i = 0; i < U; ++i) {
      t.all += w[i];
      if (at[i] < from) {
        t.sure += w[i];
        if (MIN_P && w[i] >= least) t.kept += w[i];
      }
      some |= at[i] >= from && at[i] < behind;
    }
    if (__any_sync(0xffffffffu, some)) {
#pragma unroll
      for (int i = 0; i < U; ++i)
        append(s, at[i] >= from && at[i] < behind && l[i] > row.floor_, l[i], row.lo + j + 32 * i);
    }
  }
  t.all = warp_sum64(t.all);
  t.sure = warp_sum64(t.sure);
  t.kept = MIN_P ? warp_sum64(t.kept) : t.sure;
  return t;
}

// ent[0, n) in descending order; entries differ from one another.  Long lists: bitonic; a thread has one pair
// of each step; pairs up to 32 apart stay within the 64 entries of a warp, which then needs no
// barrier with the others.
template <class Shared>
__device__ void sort_list(Shared& s, int n) {
  u64* ent = s.ent;
  if (n <= Shared::kThreads) {  // an entry's place is the number of larger ones, counted by 4, 2 or 1 threads
    const int lg = n <= Shared::kThreads / 4 ? 2 : n <= Shared::kThreads / 2 ? 1 : 0;
    __syncthreads();  // the entries are there
    const int i = threadIdx.x >> lg, part = threadIdx.x & ((1 << lg) - 1);
    const u64 e = i < n ? ent[i] : 0;
    int larger = 0;
#pragma unroll 4
    for (int j = part; j < n; j += 1 << lg) larger += ent[j] > e;
    if (lg > 0) larger += __shfl_xor_sync(0xffffffffu, larger, 1);
    if (lg > 1) larger += __shfl_xor_sync(0xffffffffu, larger, 2);
    __syncthreads();
    if (i < n && part == 0) ent[larger] = e;
    __syncthreads();
    return;
  }
  int N = 32;
  while (N < n) N <<= 1;
  for (int i = n + threadIdx.x; i < N; i += Shared::kThreads) ent[i] = 0;
  __syncthreads();
  static_assert(Shared::kList / 2 <= Shared::kThreads, "a pair for each thread");
  const int i = threadIdx.x;
  if (i < (N / 2 + 31) / 32 * 32 || N > 64) {  // whole warps; all of them where they meet at barriers
    for (int k = 2; k <= N; k <<= 1)
      for (int j = k >> 1; j > 0; j >>= 1) {
        if (i < N / 2) {
          const int a = ((i & ~(j - 1)) << 1) | (i & (j - 1)), b = a | j;
          const u64 x = ent[a], y = ent[b];
          if ((x < y) == ((a & k) == 0)) ent[a] = y, ent[b] = x;
        }
        if (j > 32 || (j == 1 && k > 32 && k < N))  // the step was or the next will be across warps
          __syncthreads();
        else
          __syncwarp();
      }
  }
  __syncthreads();
}

// pre[i] = value(0) + .. + value(i) for i < n <= 2 * Shared::kThreads.
template <class Shared, class Value>
__device__ void scan_list(Shared& s, int n, Value value) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const u64 a = 2 * tid < n ? value(2 * tid) : 0, b = 2 * tid + 1 < n ? value(2 * tid + 1) : 0;
  u64 incl = warp_scan64(a + b);
  if (n > 64) {  // else all of them are warp 0's
    if (lane == 31) s.warp64[warp] = incl;
    __syncthreads();
    const u64 v = lane < Shared::kWarps ? s.warp64[lane] : 0, sum = warp_scan64(v);
    incl += __shfl_sync(0xffffffffu, sum - v, warp);
  }
  if (2 * tid < n) s.list.pre[2 * tid] = incl - b;
  if (2 * tid + 1 < n) s.list.pre[2 * tid + 1] = incl;
  __syncthreads();
}

// The number of leading list entries whose running sum s.list.pre is below `want`.
template <class Shared>
__device__ int count_below(Shared& s, int n, u64 want) {
  const int tid = threadIdx.x;
  return __syncthreads_count(2 * tid < n && s.list.pre[2 * tid] < want) +
         __syncthreads_count(2 * tid + 1 < n && s.list.pre[2 * tid + 1] < want);
}

// The smallest entry X for which the sum of value(l, index) over the entries >= X reaches `need`, by
// radix passes over the 56 bits of an entry; for any number of entries and equal logits.
template <class Shared, class R, class Value>
__device__ u64 radix_border(cg::cluster_group& cl, Shared& s, const R& row, u64 need, Value value) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, C = (int)cl.num_blocks();
  u64 prefix = 0;
  for (int shift = 48, p = 0; shift >= 0; shift -= 8, ++p) {
    uint32_t *lo = s.hist.lo + (p & 1) * 256, *hi = s.hist.hi + (p & 1) * 256;
    cl.sync();  // the pass before last is read by all
    if (tid < 256) lo[tid] = hi[tid] = 0;
    __syncthreads();
    for (int j = tid; j < row.cnt; j += Shared::kThreads) {
      const float l = row.at(j);
      const u64 e = entry_of(l, row.lo + j);
      if (((e ^ prefix) >> 8) >> shift) continue;
      const u64 v = value(l, row.lo + j);
      if (v) add64(&lo[(e >> shift) & 255], &hi[(e >> shift) & 255], v);
    }
    cl.sync();
    if (warp == 0) {  // the digit at which the sum from above reaches `need`
      u64 v[8], sum = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e] = 0;
        for (int r = 0; r < C; ++r)
          v[e] += (u64)cl.map_shared_rank(hi, r)[255 - lane * 8 - e] << 32 |
                  cl.map_shared_rank(lo, r)[255 - lane * 8 - e];
        sum += v[e];
      }
      const u64 incl = warp_scan64(sum);
      const uint32_t hit = __ballot_sync(0xffffffffu, incl >= need);
      u64 above = incl - sum;
      if (lane == __ffs(hit) - 1) {
        int d = 0;
        bool done = false;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (!done && above + v[e] < need) above += v[e], ++d;
          else done = true;
        }
        s.border = prefix | (u64)(255 - lane * 8 - d) << shift;
        s.above = above;
      }
    }
    __syncthreads();
    prefix = s.border;
    need -= s.above;
  }
  cl.sync();  // the last pass is read by all
  return prefix;
}

template <bool IN_SHARED>
__global__ void __launch_bounds__(SP_THREADS, 2) sample_kernel(const SampleArgs a) {
  typedef SampleShared<IN_SHARED> Shared;
  constexpr int THREADS = SP_THREADS, kWarps = Shared::kWarps;
  __shared__ Shared s;
  cg::cluster_group cl = cg::this_cluster();
  const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  const int r = blockIdx.x / C, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  Row<IN_SHARED> row;
  row.lo = min(a.vocab, rank * a.slice);
  row.cnt = min(a.vocab, row.lo + a.slice) - row.lo;
  row.tab = s.tab;
  row.x = a.logits + (size_t)r * a.ld + row.lo;
  const float temp = a.temperature ? a.temperature[r] : 1.f, p = a.top_p ? a.top_p[r] : 1.f;
  const float mp = a.min_p ? a.min_p[r] : 0.f, uf = a.u[(a.step ? (size_t)*a.step * a.rows : 0) + r];
  int k = a.top_k ? a.top_k[r] : 0;

  // the row, its largest and its smallest finite logit, and whether it holds a NaN
  float hi = -INFINITY, lo = INFINITY;
  bool bad = false;
#pragma unroll (IN_SHARED ? 8 : 16)
  for (int j = tid; j < row.cnt; j += THREADS) {
    const float l = __ldg(row.x + j);
    if (IN_SHARED) shared_row[j] = l;
    hi = fmaxf(hi, l);
    if (l > -INFINITY) lo = fminf(lo, l);
    bad |= l != l;
  }
  if (tid < 16) s.tab[tid] = kExpTable[tid];
  hi = warp_max(hi);
  lo = -warp_max(-lo);
  if (lane == 0) s.warp64[warp] = (u64)__float_as_uint(hi) << 32 | __float_as_uint(lo);
  bad = __syncthreads_or(bad);
  if (tid < 32) {
    const u64 v = s.warp64[lane % kWarps];
    hi = warp_max(__uint_as_float((uint32_t)(v >> 32)));
    lo = -warp_max(-__uint_as_float((uint32_t)v));
    if (tid == 0) s.fmax = hi, s.fmin = lo, s.bad = bad;
  }
  cl.sync();
  {
    const int q = lane < C ? lane : 0;  // a block of the cluster to each lane
    hi = warp_max(*cl.map_shared_rank(&s.fmax, q));
    lo = -warp_max(-*cl.map_shared_rank(&s.fmin, q));
    bad = __any_sync(0xffffffffu, *cl.map_shared_rank(&s.bad, q));
  }
  row.lmax = hi;
  row.lmax_d = (double)hi;
  const bool greedy = temp == 0.f, ok = temp >= 0.f;
  if (bad || !ok || hi == -INFINITY) {  // the same for the whole cluster
    if (rank == 0 && tid == 0) {
      a.ids[r] = -1;
      if (a.logprob) a.logprob[r] = bad || !ok ? NAN : -INFINITY;
    }
    cl.sync();  // the other blocks have read fmax and bad
    return;
  }
  row.inv_t = greedy ? 1.0 : 1.0 / (double)temp;
  row.per_16th = row.inv_t * 23.083120654223414215;
  row.floor_ = -INFINITY;
  if (hi < INFINITY && row.inv_t > 1e-30 && row.inv_t < 1e30) {
    const float f = (float)(row.lmax_d - 32.0 / row.inv_t);
    if (f > -INFINITY && ((double)f - row.lmax_d) * row.inv_t < -31.5) row.floor_ = f;
  }
  if (greedy) k = 1;
  if (k >= a.vocab) k = 0;
  const u64 least = mp > 0.f ? (u64)ceil(fmin((double)mp, 1.0) * SP_ONE) : 0;
  const double ud = uf > 0.f ? (double)uf : 0.0;
  auto drawn = [&](u64 total) {  // the weight that the running sum has to exceed
    const double at = floor(ud * (double)total);
    return at >= (double)total || (u64)at >= total ? total - 1 : (u64)at;
  };
  auto need_of = [&](u64 total) {  // top-p: the weight that stays
    const double want = ceil((double)p * (double)total);
    return want < 1.0 ? 1ull : (u64)want;
  };

  u64 border = 0;  // entries >= border stay
  if (k > 0) {
    Buckets<Shared> bucket = {hi, 0.f};
    const float range = fminf(hi - lo, 64.f * fmaxf(1.f, greedy ? 1.f : temp));
    bucket.per = range > 0.f ? (Shared::kBuckets - 1) / range : 0.f;
    find_bucket<SP_TOKENS>(cl, s, row, bucket, [](float, int) { return (u64)1; },
                [&](u64 total) { return total < (u64)k ? total : (u64)k; });
    const int last = s.bucket;
    const u64 want = s.total < (u64)k ? s.total : (u64)k;  // tokens of -infinity never stay
    const int n = gather(cl, s, row, [&](float l, int) { return l > -INFINITY && bucket.place(l) < (float)(last + 1); });
    if (n <= Shared::kList) {  // all on the sorted list, by one block
      if (rank == 0) {
        sort_list(s, n);
        int m = (int)want;
        for (int i = tid; i < m; i += THREADS) s.list.wt[i] = row.weight(logit_of(s.ent[i]));
        __syncthreads();
        scan_list(s, m, [&](int i) { return s.list.wt[i]; });
        if (p < 1.f) m = count_below(s, m, need_of(s.list.pre[m - 1])) + 1;
        if (least)  // weights descend
          m = __syncthreads_count(2 * tid < m && s.list.wt[2 * tid] >= least) +
              __syncthreads_count(2 * tid + 1 < m && s.list.wt[2 * tid + 1] >= least);
        const u64 total = s.list.pre[m - 1], at = drawn(total);
        __syncthreads();
        // index order: entries become (index, place), inverted since the sort descends
        for (int i = tid; i < m; i += THREADS) s.ent[i] = ~((u64)index_of(s.ent[i]) << 32 | (uint32_t)i);
        sort_list(s, m);
        scan_list(s, m, [&](int i) { return s.list.wt[(uint32_t)~s.ent[i]]; });
        const int place = count_below(s, m, at + 1);
        if (tid == 0) {
          const u64 e = ~s.ent[place];
          a.ids[r] = (int)(e >> 32);
          if (a.logprob) a.logprob[r] = (float)log((double)s.list.wt[(uint32_t)e] / (double)total);
        }
      }
      cl.sync();  // block 0 has read the others' entries
      return;
    }
    cl.sync();  // the counts are read by all
    const int in_last = gather(cl, s, row, [&](float l, int) {
      return l > -INFINITY && bucket.place(l) >= (float)last && bucket.place(l) < (float)(last + 1);
    });
    if (in_last <= Shared::kList) {
      if (rank == 0) {
        sort_list(s, in_last);
        if (tid == 0) s.border = s.ent[(int)(want - s.above) - 1];
      }
      cl.sync();
      border = *cl.map_shared_rank(&s.border, 0);
      cl.sync();
    } else {
      border = radix_border(cl, s, row, want, [](float l, int) { return (u64)(l > -INFINITY); });
    }
  }
  // each warp has a part of this block's logits; what min-p lets go of for certain needs no weight
  const int part = max(32, (row.cnt + kWarps * 32 - 1) / (kWarps * 32) * 32);
  const int w0 = min(row.cnt, warp * part), w1 = min(row.cnt, w0 + part);
  const float cut = least ? (float)(row.lmax_d + (log(fmin((double)mp, 1.0)) - 1e-3) / row.inv_t) : -INFINITY;
  const float low = cut > -INFINITY ? nextafterf(cut, -INFINITY) : -INFINITY;  // (NaN and +infinity: no cut below)
  bool summed = false;
  if (p < 1.f) {
    const u64 first = border;
    Buckets<Shared> bucket = {hi, 0.f};
    const float range = fminf(hi - lo, (float)(32.1 / row.inv_t));  // beyond, no token has a weight
    bucket.per = range > 0.f ? (Shared::kBuckets - 1) / range : 0.f;
    // the border by the entries of block 0's list, of which the running sum before them is `above`; 0 if
    // it is not among them
    auto border_of_list = [&](int n, u64 above, u64 want) {
      if (rank == 0) {
        sort_list(s, n);
        for (int i = tid; i < n; i += THREADS) s.list.wt[i] = row.weight(logit_of(s.ent[i]));
        __syncthreads();
        scan_list(s, n, [&](int i) { return s.list.wt[i]; });
        const int place = above < want ? count_below(s, n, want - above) : n;
        if (tid == 0) s.border = place < n ? s.ent[place] : 0;
      }
      cl.sync();
      return *cl.map_shared_rank(&s.border, 0);
    };
    // those of the list that stay and lie in this block join their warp's sum
    auto add_list = [&](int n) {
      const int own = rank == 0 ? n : s.n;
      for (int i = tid; i < own; i += THREADS) {
        const u64 e = s.ent[i];
        const int j = index_of(e) - row.lo;
        if (e < border || j < 0 || j >= row.cnt) continue;
        const u64 w = row.weight(logit_of(e));
        if (w && w >= least) add64(&s.part_lo[j / part], &s.part_hi[j / part], w);
      }
      __syncthreads();
    };
    const bool plain = first == 0 && row.floor_ > -INFINITY && bucket.per > 0.f && bucket.per < 1e30f;
    if (plain && a.slice >= SP_MIDDLE_SLICE) {
      // The bucket by middles, which may be off by one where the border lies near its end; then the
      // exact sums and a list of the bucket and that neighbour, each token's weight computed once (256
      // rows of 151643 tokens 288 -> 240 us, 64 rows of 73448 41 -> 37; slices of 9181 tokens gain
      // nothing, 8 rows of 73448 with mixed settings 23.5 -> 24.3).
      find_bucket<SP_MIDDLES>(cl, s, row, bucket, [](float, int) { return (u64)0; }, need_of);
      const float from = (float)max(0, s.bucket - (s.into < 0.25f)), behind = (float)(s.bucket + 1 + (s.into > 0.75f));
      if (tid == 0) s.n = 0;
      __syncthreads();
      const Sums t = least ? sum_all<true>(s, row, bucket, w0, w1, from, behind, least)
                           : sum_all<false>(s, row, bucket, w0, w1, from, behind, least);
      if (lane == 0) {
        s.warp64[warp] = t.all;
        s.warp_sure[warp] = t.sure;
        s.part_lo[warp] = (uint32_t)t.kept;
        s.part_hi[warp] = (uint32_t)(t.kept >> 32);
      }
      __syncthreads();
      if (warp == 0) {
        const u64 all = warp_sum64(lane < kWarps ? s.warp64[lane] : 0);
        const u64 sure = warp_sum64(lane < kWarps ? s.warp_sure[lane] : 0);
        if (lane == 0) s.total = all, s.above = sure;
      }
      const int n = collect(cl, s);
      const u64 total = warp_sum64(lane < C ? *cl.map_shared_rank(&s.total, lane) : 0);
      const u64 sure = warp_sum64(lane < C ? *cl.map_shared_rank(&s.above, lane) : 0);
      if (n > 0 && n <= Shared::kList) border = border_of_list(n, sure, need_of(total));
      if (border) {
        add_list(n);
        summed = true;
      } else {
        cl.sync();  // the other blocks have read total, above and border
      }
    }
    if (!summed) {
      auto weight = [&](float l, int i) { return first == 0 || entry_of(l, i) >= first ? row.weight(l) : (u64)0; };
      if (plain)
        find_bucket<SP_PLAIN>(cl, s, row, bucket, [](float, int) { return (u64)0; }, need_of);
      else
        find_bucket<SP_WEIGHTS>(cl, s, row, bucket, weight, need_of);
      const float last = (float)s.bucket, next = last + 1.f;
      const u64 want = need_of(s.total), above = s.above;
      // before the border's bucket all stay; the bucket's own go on the list
      if (tid == 0) s.n = 0;
      __syncthreads();
      const u64 sure = plain ? sum_kept(s, row, w0, w1, least, [&](float l, int j) {
        const float at = (bucket.lmax - l) * bucket.per;
        append(s, l > row.floor_ && at >= last && at < next, l, row.lo + j);
        return at < last && l >= low;
      }) : sum_kept(s, row, w0, w1, least, [&](float l, int j) {
        const float at = bucket.place(l);
        const bool in = j < w1 && (first == 0 || entry_of(l, row.lo + j) >= first);
        append(s, in && at >= last && at < next, l, row.lo + j);
        return in && at < last && l >= low;
      });
      if (lane == 0) s.part_lo[warp] = (uint32_t)sure, s.part_hi[warp] = (uint32_t)(sure >> 32);
      const int n = collect(cl, s);
      if (n <= Shared::kList) {
        border = border_of_list(n, above, want);
        add_list(n);
        summed = true;
      } else {
        border = radix_border(cl, s, row, want, weight);
      }
    }
  }

  // the sums of the warps' parts, then the warp that holds the token walks its part
  const float edge = border ? logit_of(border) : -INFINITY;
  const int edge_index = border ? index_of(border) : a.vocab;
  auto stays = [&](float l, int j) {
    return (l > edge || (l == edge && row.lo + j <= edge_index)) && l >= low;
  };
  u64 sum;
  if (summed) {
    sum = (u64)s.part_hi[warp] << 32 | s.part_lo[warp];
  } else {
    sum = sum_kept(s, row, w0, w1, least, stays);
  }
  if (lane == 0) s.warp64[warp] = sum;
  __syncthreads();
  u64 before = 0;
  {
    const u64 v = lane < kWarps ? s.warp64[lane] : 0;
    const u64 incl = warp_scan64(v);
    before = __shfl_sync(0xffffffffu, incl - v, warp);
    if (tid == 31) s.block_sum = incl;
  }
  cl.sync();
  const u64 block_sum = lane < C ? *cl.map_shared_rank(&s.block_sum, lane) : 0;
  const u64 block_incl = warp_scan64(block_sum);
  const u64 total = __shfl_sync(0xffffffffu, block_incl, 31), at = drawn(total);
  before += __shfl_sync(0xffffffffu, block_incl - block_sum, rank);
  if (tid == 0) s.n = -1;
  __syncthreads();
  if (lane == 0 && before <= at && at < before + sum) {
    s.n = warp;
    s.run = before;
  }
  __syncthreads();
  if (s.n >= 0) {  // one block of the cluster: all its warps walk the part of that warp
    u64 run = s.run;
    const int j0 = s.n * part, j1 = min(row.cnt, j0 + part);
    float next = j0 + tid < j1 ? row.at(j0 + tid) : 0.f;
    for (int j = j0 + tid; j - tid < j1; j += THREADS) {
      const float l = next;
      if (j + THREADS < j1) next = row.at(j + THREADS);
      u64 w = j < j1 && stays(l, j) ? row.weight(l) : 0;
      if (w < least) w = 0;
      u64 incl = warp_scan64(w);
      __syncthreads();  // warp64 of the round before is read
      if (lane == 31) s.warp64[warp] = incl;
      __syncthreads();
      for (int q = 0; q < kWarps; ++q) {
        if (q == warp) incl += run;
        run += s.warp64[q];
      }
      if (incl - w <= at && at < incl) {
        a.ids[r] = row.lo + j;
        if (a.logprob) a.logprob[r] = (float)log((double)w / (double)total);
      }
      if (run > at) break;
    }
  }
  cl.sync();  // the other blocks have read this one's sum
}

// Blocks of a row, and whether they hold it in shared memory.
struct SampleShape {
  int blocks;
  bool in_shared;
};
constexpr int SP_SLICE = 32768;  // logits of a block in shared memory at most: 128 KB
constexpr int SP_TWO = 18432;    // that leave room for two blocks on an SM
// As many blocks of a row as there are SMs for (one row of 73448 tokens: 8 blocks 15 us, 2 blocks
// 27 us; 64 rows: 4 blocks 43 us, 8 blocks 57 us).  256 rows of 151643 tokens that are read from L2: 1
// block 252 us, 2 232, 4 249, 8 381; 8 with the row in shared memory 345 us (2 blocks by now: 183).
SampleShape shape_of(int rows, int vocab) {
  SampleShape p = {1, true};
  while (p.blocks < SP_MAX_CLUSTER && vocab > 2048 * p.blocks && rows * p.blocks < 148) p.blocks *= 2;
  const int slice = (vocab + p.blocks - 1) / p.blocks;
  p.in_shared = slice <= SP_TWO || (slice <= SP_SLICE && rows * p.blocks <= 148);
  if (!p.in_shared && p.blocks == 1) p.blocks = 2;
  return p;
}

}  // namespace

cudaError_t sample_configure() {
  return cudaFuncSetAttribute(sample_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, SP_SLICE * 4);
}

cudaError_t launch_sample(const float* logits, int64_t row_stride, int rows, int vocab, const float* u, const int* step,
                          const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                          int32_t* ids, float* logprob, cudaStream_t st) {
  if (rows <= 0 || vocab <= 0 || vocab > SP_MAX_VOCAB) return cudaErrorInvalidValue;
  const SampleShape p = shape_of(rows, vocab);
  SampleArgs a = {logits, row_stride, rows, vocab, (vocab + p.blocks - 1) / p.blocks, u, step, temperature, top_k,
                  top_p, min_p, ids, logprob};
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(rows * p.blocks);
  cfg.blockDim = dim3(SP_THREADS);
  cfg.dynamicSmemBytes = p.in_shared ? (size_t)a.slice * 4 : 0;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.blocks;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  count_launch();
  return p.in_shared ? cudaLaunchKernelEx(&cfg, sample_kernel<true>, a)
                     : cudaLaunchKernelEx(&cfg, sample_kernel<false>, a);
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
  if (row_stride < 0) return fail(ctx, VX_ERR_SHAPE, "sample: negative row stride");
  if (rows == 0) return VX_OK;
  DeviceGuard guard(ctx->device);
  VX_CUDA(ctx, launch_sample(logits, row_stride, rows, vocab, u, nullptr, temperature, top_k, top_p, min_p, ids, logprob,
                             pick_stream(ctx, stream)));
  return VX_OK;
}
