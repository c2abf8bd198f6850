// kq_sample.cu -- the next token of every sequence from its logits
// (include/pesti_decoder.h, kq_dec_sample): temperature, top-k, top-p, min-p and
// the draw from a given random number.
//
// Mathematics: in the order (logit descending, index ascending) each filter
// keeps a prefix, so every one is a cut at one token of that order.  The weights
// 2^((z - max) log2 e / T) are 64-bit fixed point, 2^44 or less for the largest:
// their sums are exact whatever their order, and a draw next to the border of
// two tokens falls on the same side on every run.
//
// What bounds it: one read of the logits from HBM, and where the weights of the
// whole vocabulary are summed 8 FP64 instructions (of some 25) each.  A cluster
// of up to eight CTAs shares a row: every CTA keeps its slice of the logits in
// shared memory, so they are read once, and what the slices know of one another
// goes over distributed shared memory.
//  * top-k: the k-th greatest of one CTA's per-thread maxima lies no higher than
//    the k-th token; the candidates from the highest such bound up (a few times
//    k) go to one CTA, which ranks them against one another and applies the other
//    filters to them;
//  * top-p over more than that: weights in 2048 bins of the distance from the
//    maximum, then the bin of the border: its tokens are ranked by one CTA where
//    they are few, else the bins are refined over the 64-bit words (key of the
//    logit, ~index) themselves, 11 bits at a time;
//  * the draw: sums per thread over consecutive tokens, and one thread walks the
//    stretch that holds it.
// Measured: one row of 151,936 with every filter 11.7 us, 32 rows of 128,256 under
// top-p 38.1 us (issue slots 49% busy: 139 warp instructions per 32 tokens, 60 of
// them for the shared atomics of the bins; one read of the logits would take 2.5), 64 rows of 151,936 with settings of their own 55.0 us.
#include "kq_common.cuh"
#include "kq_kernels.h"

#include <cooperative_groups.h>
#include <float.h>
#include <math.h>

namespace kq {
namespace {

namespace cg = cooperative_groups;
typedef unsigned long long u64;

constexpr int SM_MAX_WARPS = 32;
constexpr int SM_BINS = 2048;
constexpr int SM_LIST = 1024;  // candidates one CTA ranks
constexpr int SM_MAX_CLUSTER = 8;
constexpr int SM_SLICE = SAMPLE_MAX_VOCAB / SM_MAX_CLUSTER;  // logits a CTA can hold
constexpr int SM_POW = 256;  // (2^8 entries of 2^20 / 2^8 in a double's upper half: the shift by 12 below)
constexpr int SM_FRAC = 44;  // distances above 31.2 T weigh less than 1/2: 0

// f32 -> unsigned with the same order (-0 as 0)
__device__ __forceinline__ uint32_t order_key(float f) {
  const uint32_t u = __float_as_uint(f + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_logit(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
// a token's word: greater is earlier in the order
__device__ __forceinline__ u64 word_of(float z, int i) { return (u64)order_key(z) << 32 | (uint32_t)~i; }
__device__ __forceinline__ float word_logit(u64 w) { return key_logit((uint32_t)(w >> 32)); }
__device__ __forceinline__ int word_index(u64 w) { return (int)~(uint32_t)w; }

// The last token that stays: those before it in the order do too.  A token stays
// where its logit is at least `z` (up to index i) or `above`, the next number (from
// there on): one comparison each, the choice for four neighbours at once.
struct Cut {
  float z, above;
  int i;
  __device__ __forceinline__ Cut(float z_, int i_) : z(z_), above(nextafterf(z_, INFINITY)), i(i_) {}
  __device__ __forceinline__ bool keeps(float f, int at) const { return f >= (at <= i ? z : above); }
  __device__ __forceinline__ void keeps4(const float (&f)[4], int at, bool (&stay)[4]) const {
    const float least = at + 3 <= i ? z : above;
#pragma unroll
    for (int q = 0; q < 4; ++q) stay[q] = f[q] >= least;
    if ((unsigned)(i - at) < 3u) {  // the border lies among the four
#pragma unroll
      for (int q = 0; q < 4; ++q) stay[q] = keeps(f[q], at + q);
    }
  }
};

struct SampleShared {
  double pow2[SM_POW];  // 2^(frac + i / SM_POW)
  u64 sums[SM_MAX_WARPS];
  u64 tot[2][SM_MAX_CLUSTER], tot2[2][SM_MAX_CLUSTER];  // two values of every CTA of the cluster, two sets in turn
  u64 res[4];                                     // what this CTA found for all
  unsigned listed;                                // first CTA: candidates so far
  int first;                                      // the first index of the greatest logit
  float kth[2];  // the K-th greatest of the threads' own, and the ceil(K / CTAs)-th
  uint32_t lo[SM_BINS], hi[SM_BINS];   // histogram, 64-bit sums as two words
  u64 list[SM_LIST], weight[SM_LIST];  // first CTA: candidates
};
static_assert(sizeof(SampleShared) % 16 == 0, "the slice follows");
// The CTA's shared memory: this, then its slice of the logits, padded with -inf.
// (Named where it is used, so that every access is known to be one to shared memory.)
extern __shared__ __align__(16) uint8_t sample_smem[];
__device__ __forceinline__ SampleShared& shared() { return *reinterpret_cast<SampleShared*>(sample_smem); }
__device__ __forceinline__ float* slice_logits() { return reinterpret_cast<float*>(sample_smem + sizeof(SampleShared)); }

// Exclusive sum over the block's NT threads; `total` gets the sum.
template <int NT>
__device__ __forceinline__ u64 block_scan(u64 v, u64* sums, u64& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto scan = [&](u64 x) {  // inclusive, over the warp
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    return x;
  };
  const u64 x = scan(v);
  __syncthreads();
  if (lane == 31) sums[warp] = x;
  __syncthreads();
  const u64 w = lane < NT / 32 ? sums[lane] : 0, upto = scan(w);
  total = __shfl_sync(0xffffffffu, upto, 31);
  return __shfl_sync(0xffffffffu, upto - w, warp) + x - v;
}

// The weights of one row.
struct Weights {
  double c, zmax64;         // SM_POW log2 e / T, the greatest logit
  float zmax, per_t, zero;  // the greatest logit, 128 / T, a logit from which on the weight is 0
  const double* pow2;       // 2^(frac + i / SM_POW)
  __device__ __forceinline__ Weights(float top, float T, const double* table)
      : c(SM_POW * 1.4426950408889634074 / (double)T), zmax64((double)top), zmax(top), per_t(fminf(128.f / T, FLT_MAX)),
        zero(nextafterf(top - 31.6f * T, -INFINITY)), pow2(table) {
    // Where the logits' steps are far above T (31.6 T below the top is one step), every token below the
    // top weighs 0: its distance is kept to what the exponent holds.
    const double most = 46.0 * SM_POW, t = (zmax64 - (double)fmaxf(zero, -FLT_MAX)) * c;
    if (t > most) c *= most / t;
  }
  // the bin of the distance from the maximum, 128 per T; the last takes all beyond
  __device__ __forceinline__ int bin(float f) const { return (int)fminf((zmax - f) * per_t, (float)(SM_BINS - 1)); }
  // The weight is e p to about 2e-13: 2^t = 2^(n / 256) 2^r with |r| <= 1/512, a
  // table and the exponential series in r.
  __device__ __forceinline__ void parts(float z, double& e, double& p) const {
    constexpr double ROUND = 6755399441055744.0;  // 1.5 2^52: the sum's last bits are the nearest integer
    const double d = (double)fmaxf(z, zero) - zmax64;
    const double nd = fma(d, c, ROUND);
    const double r = fma(d, c, ROUND - nd);
    const int n = __double2loint(nd);
    constexpr double A = 0.69314718055994530942 / SM_POW;
    p = fma(r, fma(r, fma(r, A * A * A / 6, A * A / 2), A), 1.0);
    const double w = pow2[n & (SM_POW - 1)];
    e = __hiloint2double(__double2hiint(w) + (int)((uint32_t)(n & ~(SM_POW - 1)) << 12), __double2loint(w));
  }
  __device__ __forceinline__ double scaled(float z) const {
    double e, p;
    parts(z, e, p);
    return e * p;
  }
  // The weight rounded to an integer, plus ONE: the bits of 2^52 + weight.
  static constexpr u64 ONE = 0x4330000000000000ull;
  __device__ __forceinline__ u64 biased(float z) const {
    double e, p;
    parts(z, e, p);
    return (u64)__double_as_longlong(fma(e, p, 4503599627370496.0));
  }
  __device__ __forceinline__ u64 fixed(float z) const { return biased(z) - ONE; }
  // The least logit whose weight is `share` (in (0, 1]) of the greatest: near the
  // logarithm, the last steps by the definition.
  __device__ __forceinline__ float logit_of(double share, double T) const {
    auto stays = [&](float z) { return exp(((double)z - zmax64) / T) >= share; };
    float z = (float)fmax(zmax64 + T * log(share), -(double)FLT_MAX);
    for (int k = 0; k < 64 && !stays(z); ++k) z = nextafterf(z, INFINITY);
    for (int k = 0; k < 64; ++k) {
      const float y = nextafterf(z, -INFINITY);
      if (y == -INFINITY || !stays(y)) break;
      z = y;
    }
    return z;
  }
};

// One row's CTAs of NT threads: their slice and what they share.
template <int NT>
struct Row {
  cg::cluster_group cluster;
  int CL, rank, i0, n;
  int turn = 0;  // the set of shared().tot published last

  // f(z[4], first index) over the slice, four consecutive tokens at a time
  template <class F>
  __device__ __forceinline__ void each4(F f) {
    for (int i = 4 * threadIdx.x; i < n; i += 4 * NT) {
      const float4 v = *reinterpret_cast<const float4*>(slice_logits() + i);
      const float a[4] = {v.x, v.y, v.z, v.w};
      f(a, i0 + i);
    }
  }

  // Two values of every CTA known to all.  (Two sets in turn: the last one may
  // still be read in another CTA while this one is written.)
  __device__ __forceinline__ void publish(u64 a, u64 b) {
    turn ^= 1;
    if (threadIdx.x < CL) {
      SampleShared* to = cluster.map_shared_rank(&shared(), threadIdx.x);
      to->tot[turn][rank] = a;
      to->tot2[turn][rank] = b;
    }
    cluster.sync();
  }
  __device__ __forceinline__ u64 tot(int r) const { return shared().tot[turn][r]; }
  __device__ __forceinline__ u64 tot2(int r) const { return shared().tot2[turn][r]; }

  // The bins filled with measure(z): bins_of(z[4], first index, bins[4]) says where
  // (-1: left out).
  template <class Bins, class Measure>
  __device__ void fill_bins(Bins bins_of, Measure measure) {
    for (int e = threadIdx.x; e < SM_BINS; e += NT) shared().lo[e] = shared().hi[e] = 0;
    __syncthreads();
    each4([&](const float (&v)[4], int i) {
      int k[4];
      u64 m[4];
      uint32_t old[4];
      bins_of(v, i, k);
#pragma unroll
      for (int q = 0; q < 4; ++q) m[q] = measure(v[q]);
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (k[q] >= 0) old[q] = atomicAdd(&shared().lo[k[q]], (uint32_t)m[q]);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if (k[q] < 0) continue;
        const uint32_t h = (uint32_t)(m[q] >> 32) + (old[q] + (uint32_t)m[q] < old[q]);  // the carry
        if (h) atomicAdd(&shared().hi[k[q]], h);
      }
    });
  }

  // From all slices' bins: the bin in which the running sum from bin 0 reaches
  // target(total), and how much of that bin it takes (`left`).  False where it is
  // not reached.  A cluster.sync() must follow before the CTA ends.
  template <class Target>
  __device__ bool find_bin(Target target_of, int& bin, u64& left) {
    cluster.sync();
    const int bins = SM_BINS / CL, per = (bins + NT - 1) / NT;  // this CTA joins bins [rank bins, ..)
    constexpr int MOST = SM_BINS / NT;
    u64 m[MOST], sum = 0;
#pragma unroll
    for (int q = 0; q < MOST; ++q) {
      m[q] = 0;
      const int e = threadIdx.x * per + q;
      if (q < per && e < bins) {
        uint32_t lo[SM_MAX_CLUSTER], hi[SM_MAX_CLUSTER];
#pragma unroll
        for (int r = 0; r < SM_MAX_CLUSTER; ++r) {
          const SampleShared* from = cluster.map_shared_rank(&shared(), r < CL ? r : 0);
          lo[r] = r < CL ? from->lo[rank * bins + e] : 0;
          hi[r] = r < CL ? from->hi[rank * bins + e] : 0;
        }
#pragma unroll
        for (int r = 0; r < SM_MAX_CLUSTER; ++r) m[q] += (u64)hi[r] << 32 | lo[r];
      }
      sum += m[q];
    }
    u64 total;
    u64 before = block_scan<NT>(sum, shared().sums, total);
    publish(total, 0);
    u64 all = 0, start = 0;
    for (int r = 0; r < CL; ++r) {
      if (r < rank) start += tot(r);
      all += tot(r);
    }
    const u64 target = target_of(all);
    if (target > all) return false;
    before += start;
#pragma unroll
    for (int q = 0; q < MOST; ++q) {
      if (target > before && target <= before + m[q]) {
        shared().res[0] = (u64)(rank * bins + threadIdx.x * per + q);
        shared().res[1] = target - before;
      }
      before += m[q];
    }
    int owner = 0;
    for (u64 sofar = tot(0); sofar < target; sofar += tot(owner)) ++owner;
    cluster.sync();
    const SampleShared* from = cluster.map_shared_rank(&shared(), owner);
    bin = (int)from->res[0];
    left = from->res[1];
    return true;
  }

  // The tokens of pred(z, index) to the first CTA's list, counted there (what does
  // not fit is dropped); their number.  A cluster.sync() must follow before the
  // CTA ends.
  template <class Pred>
  __device__ unsigned gather(Pred pred) {
    SampleShared* first = cluster.map_shared_rank(&shared(), 0);
    each4([&](const float (&v)[4], int i) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if (!pred(v[q], i + q)) continue;
        const unsigned at = atomicAdd(&first->listed, 1u);
        if (at < SM_LIST) first->list[at] = word_of(v[q], i + q);
      }
    });
    cluster.sync();
    return first->listed;
  }

  // The token at which the running sum of measure(z), over the tokens of pred in
  // order, reaches `left` (their sum is at least that).
  template <class Measure, class Pred>
  __device__ __forceinline__ Cut border(Measure measure, u64 left, Pred pred) {
    const unsigned listed = gather(pred);
    if (listed <= SM_LIST) {
      if (rank == 0) {
        for (unsigned e = threadIdx.x; e < listed; e += NT) shared().weight[e] = measure(word_logit(shared().list[e]));
        __syncthreads();
        for (unsigned e = threadIdx.x; e < listed; e += NT) {
          const u64 w = shared().list[e];
          u64 before = 0;
          for (unsigned j = 0; j < listed; ++j) before += shared().list[j] > w ? shared().weight[j] : 0;
          if (before < left && left <= before + shared().weight[e]) shared().res[2] = w;
        }
      }
      cluster.sync();
      const u64 w = cluster.map_shared_rank(&shared(), 0)->res[2];
      if (rank == 0 && threadIdx.x == 0) shared().listed = 0;
      return Cut(word_logit(w), word_index(w));
    }
    const Refined r = refine(*this, measure, left, pred);
    turn = r.turn;
    return r.cut;
  }

  // The same where too many tokens satisfy pred: refined over the words, from
  // their exact range.  (A call of its own: seldom needed, and it would hold
  // registers.)
  struct Refined {
    Cut cut;
    int turn;
  };
  template <class Measure, class Pred>
  __device__ static __noinline__ Refined refine(Row R, Measure measure, u64 left, Pred pred) { return R.refined(measure, left, pred); }
  template <class Measure, class Pred>
  __device__ __forceinline__ Refined refined(Measure measure, u64 left, Pred pred) {
    u64 low = ~0ull, high = 0;
    each4([&](const float (&v)[4], int i) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if (!pred(v[q], i + q)) continue;
        const u64 w = word_of(v[q], i + q);
        low = w < low ? w : low;
        high = w > high ? w : high;
      }
    });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const u64 a = __shfl_xor_sync(0xffffffffu, low, o), c = __shfl_xor_sync(0xffffffffu, high, o);
      low = a < low ? a : low;
      high = c > high ? c : high;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) {
      shared().list[threadIdx.x >> 5] = low;
      shared().weight[threadIdx.x >> 5] = high;
    }
    __syncthreads();
    for (int w = 0; w < NT / 32; ++w) {
      low = shared().list[w] < low ? shared().list[w] : low;
      high = shared().weight[w] > high ? shared().weight[w] : high;
    }
    publish(low, high);
    if (rank == 0 && threadIdx.x == 0) shared().listed = 0;
    for (int r = 0; r < CL; ++r) {
      low = tot(r) < low ? tot(r) : low;
      high = tot2(r) > high ? tot2(r) : high;
    }
    while (low < high) {
      const int shift = max(0, 64 - __clzll((long long)(high - low)) - 11);
      int bin = 0;
      const u64 goal = left;
      fill_bins(
          [&](const float (&v)[4], int i, int (&k)[4]) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const u64 w = word_of(v[q], i + q);
              k[q] = w >= low && w <= high && pred(v[q], i + q) ? SM_BINS - 1 - (int)((w - low) >> shift) : -1;
            }
          },
          measure);
      find_bin([&](u64) { return goal; }, bin, left);
      low += (u64)(SM_BINS - 1 - bin) << shift;
      const u64 top = low + ((1ull << shift) - 1);
      high = top < high ? top : high;
    }
    return Refined{Cut(word_logit(low), word_index(low)), turn};
  }
};

// What a row's first CTA does alone: `m` candidates in S.list hold the first K <=
// NT tokens; top-p, min-p (logits from `least` up) and the draw among those.
template <int NT, class Answer>
__device__ __noinline__ void draw_from_list(Weights W, int m, int K, double P, float least, double U,
                                            Answer answer) {
  SampleShared& S = shared();
  const int tid = threadIdx.x;
  for (int e = tid; e < m; e += NT) {  // into their order
    const u64 w = S.list[e];
    int place = 0;
    for (int j = 0; j < m; ++j) place += S.list[j] > w;
    if (place < K) S.weight[place] = w;
  }
  __syncthreads();
  const u64 mine = tid < K ? S.weight[tid] : 0;
  const float z = word_logit(mine);
  u64 w = tid < K ? W.fixed(z) : 0, total;
  u64 before = block_scan<NT>(w, S.sums, total);
  const bool stay = tid < K && (tid == 0 || ((!(P < 1.0) || (double)before < ceil(P * (double)total)) && z >= least));
  if (!stay) w = 0;
  const int kept = __syncthreads_count(stay);
  block_scan<NT>(w, S.sums, total);
  if (stay) S.list[tid] = w;
  __syncthreads();
  if (!stay) return;
  const double t = U * (double)total;
  const u64 goal = t > 0.0 ? min((u64)t, total - 1) : 0;
  before = 0;  // a lower index has a greater low half of the word
  for (int j = 0; j < kept; ++j) before += (uint32_t)S.weight[j] > (uint32_t)mine ? S.list[j] : 0;
  if (before <= goal && goal < before + w) answer(word_index(mine), (float)(W.scaled(z) / (double)total), kept);
}

// NT 512: two CTAs per SM; 1024: one
template <int NT>
__global__ void __launch_bounds__(NT, 1024 / NT) sample_kernel(const SampleArgs A, int slice, int frac) {
  SampleShared& S = shared();
  cg::cluster_group cluster = cg::this_cluster();
  const int CL = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int64_t b = blockIdx.x / CL;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int i0 = min(A.vocab, rank * slice), n = min(A.vocab, i0 + slice) - i0;  // this CTA's tokens
  float* z = slice_logits();
  Row<NT> R{cluster, CL, rank, i0, n};
  cluster.barrier_arrive();  // this CTA has started
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (tid < 16) {  // 2^(i / 256) = 2^(16 a / 256) 2^(b / 256)
    S.pow2[16 * tid] = exp2(frac + tid / 16.0);
    if (tid) S.pow2[tid] = exp2(frac + tid / 256.0);
  }
  if (tid == 0) S.listed = 0;
  if (tid < 8) z[n + tid] = -INFINITY;
  for (int e = tid; e < SM_BINS; e += NT) S.lo[e] = 0;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // the slice into shared memory, 16 bytes a copy where the row allows it
  const float* row = A.logits + b * A.ld + i0;
  const int quads = (reinterpret_cast<uintptr_t>(row) & 15) == 0 ? n / 4 : 0;
  for (int i = tid; i < quads; i += NT)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(z + 4 * i)),
                 "l"(row + 4 * i)
                 : "memory");
  for (int i = 4 * quads + tid; i < n; i += NT)
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"((uint32_t)__cvta_generic_to_shared(z + i)),
                 "l"(row + i)
                 : "memory");
  asm volatile("cp.async.commit_group;" ::: "memory");
  const float T = A.temperature ? A.temperature[b] : 1.f;
  const int K = A.top_k ? A.top_k[b] : 0;
  const double P = A.top_p ? (double)A.top_p[b] : 1.0, M = A.min_p ? (double)A.min_p[b] : 0.0;
  const double U = (double)A.u[b];
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
  if (tid >= 16 && tid < SM_POW && tid % 16)
    S.pow2[tid] = S.pow2[tid & ~15] * S.pow2[tid & 15] * __hiloint2double((1023 - frac) << 20, 0);

  // ---- the greatest logit of the slice, and bounds from below for the K-th: order
  // statistics of the threads' own greatest, by bins of 1/64 ----
  float own = -INFINITY;  // (NaN never is the greater one)
  R.each4([&](const float (&v)[4], int) {
    own = fmaxf(own, fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])));
  });
  float top = own;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) reinterpret_cast<float*>(S.sums)[warp] = top;
  if (tid == 0) S.kth[0] = S.kth[1] = -INFINITY;
  __syncthreads();
  for (int w = 0; w < NT / 32; ++w) top = fmaxf(top, reinterpret_cast<float*>(S.sums)[w]);
  if (K > 1 && K <= NT) {
    const float q = (top - own) * 64.f;  // (inf or NaN where there is nothing)
    const int k = q < (float)SM_BINS ? (int)q : -1;
    if (k >= 0) atomicAdd(&S.lo[k], 1u);
    __syncthreads();
    constexpr int PER = SM_BINS / NT;
    u64 m[PER], sum = 0, all;
#pragma unroll
    for (int e = 0; e < PER; ++e) sum += m[e] = S.lo[PER * tid + e];
    u64 before = block_scan<NT>(sum, S.sums, all);
    const u64 want[2] = {(u64)K, (u64)((K + CL - 1) / CL)};
#pragma unroll
    for (int e = 0; e < PER; ++e) {
#pragma unroll
      for (int k = 0; k < 2; ++k)
        // the bin's lower edge, and a little less: what rounding leaves of the distance
        if (before < want[k] && want[k] <= before + m[e])
          S.kth[k] = top - (PER * tid + e + 1) / 64.f - 1e-5f * (1.f + fabsf(top));
      before += m[e];
    }
    __syncthreads();
  }
  cluster.barrier_wait();  // every CTA has started: its shared memory may be written
  R.publish(__float_as_uint(top), (u64)__float_as_uint(S.kth[0]) << 32 | __float_as_uint(S.kth[1]));
  // at least K tokens lie above the K-th of any CTA, and above the least of the ceil(K / CTAs)-th
  float kth = -INFINITY, share = INFINITY;
  for (int r = 0; r < CL; ++r) {
    top = fmaxf(top, __uint_as_float((uint32_t)R.tot(r)));
    kth = fmaxf(kth, __uint_as_float((uint32_t)(R.tot2(r) >> 32)));
    share = fminf(share, __uint_as_float((uint32_t)R.tot2(r)));
  }
  kth = fmaxf(kth, share);
  auto answer = [&](int token, float prob, int kept) {
    A.tokens[b] = token;
    if (A.prob) A.prob[b] = prob;
    if (A.kept) A.kept[b] = kept;
  };
  if (top == -INFINITY) {  // no token is possible
    if (rank == 0 && tid == 0) answer(-1, 0.f, 0);
    return;
  }
  if (!(T > 0.f) || K == 1 || !(P > 0.0) || !(M <= 1.0)) {  // the first token alone stays
    if (tid == 0) S.first = INT_MAX;
    __syncthreads();
    R.each4([&](const float (&v)[4], int i) {
#pragma unroll
      for (int q = 3; q >= 0; --q)
        if (v[q] == top) atomicMin(&S.first, i + q);
    });
    __syncthreads();
    R.publish((u64)S.first, 0);
    u64 first = INT_MAX;
    for (int r = 0; r < CL; ++r) first = R.tot(r) < first ? R.tot(r) : first;
    if (rank == 0 && tid == 0) answer((int)first, 1.f, 1);
    return;
  }
  const bool endless = top == INFINITY;
  if (endless) {  // only tokens of +inf carry weight: 0 for them, the least number for the others
    for (int i = tid; i < n; i += NT)
      z[i] = z[i] == INFINITY ? 0.f : z[i] > -INFINITY ? -FLT_MAX : -INFINITY;
    top = 0.f;
    __syncthreads();
  }
  const Weights W(top, T, S.pow2);
  // min-p: the least logit that stays
  const float least = M > 0.0 ? W.logit_of(M, (double)T) : -INFINITY;
  auto fixed = [W](float f) { return W.fixed(f); };
  auto one = [](float) { return (u64)1; };

  Cut cut(-INFINITY, -1);
  if (K > 0) {
    if (kth > -INFINITY && !endless) {
      const unsigned listed = R.gather([&](float f, int) { return f >= kth; });
      cluster.sync();
      if (listed <= SM_LIST) {
        if (rank == 0) draw_from_list<NT>(W, (int)listed, K, P, least, U, answer);
        return;
      }
      if (rank == 0 && tid == 0) S.listed = 0;
    }
    // too many candidates (a large K, or many tokens of one value): the K-th token itself
    auto near = [top](float f) {
      const float q = (top - f) * 64.f;
      return q < (float)SM_BINS ? (int)q : -1;
    };
    int bin = 0;
    u64 left = 0;
    R.fill_bins(
        [&](const float (&v)[4], int, int (&k)[4]) {
#pragma unroll
          for (int q = 0; q < 4; ++q) k[q] = near(v[q]);
        },
        one);
    if (R.find_bin([&](u64) { return (u64)K; }, bin, left)) {
      cut = R.border(one, left, [near, bin](float f, int) { return near(f) == bin; });
    } else {
      u64 able = 0;
      R.each4([&](const float (&v)[4], int) {
#pragma unroll
        for (int q = 0; q < 4; ++q) able += v[q] > -INFINITY;
      });
      block_scan<NT>(able, S.sums, able);
      R.publish(able, 0);
      able = 0;
      for (int r = 0; r < CL; ++r) able += R.tot(r);
      if ((u64)K < able) cut = R.border(one, (u64)K, [](float f, int) { return f > -INFINITY; });
    }
  }
  if (P < 1.0) {
    int bin = 0;
    u64 left = 0;
    const Cut first_k = cut;
    R.fill_bins(
        [&](const float (&v)[4], int i, int (&k)[4]) {
          bool stay[4];
          first_k.keeps4(v, i, stay);
#pragma unroll
          for (int q = 0; q < 4; ++q) k[q] = stay[q] ? W.bin(v[q]) : -1;
        },
        fixed);
    R.find_bin([&](u64 all) { return min(max((u64)ceil(P * (double)all), 1ull), all); }, bin, left);
    cut = R.border(fixed, left, [W, bin, first_k](float f, int i) { return W.bin(f) == bin && first_k.keeps(f, i); });
  }

  if (least > cut.z) cut = Cut(least, INT_MAX);

  // ---- the draw: thread t sums the quads [t c, (t + 1) c) of the slice (c odd: no bank is hit twice) ----
  const int quads_here = (n + 3) / 4, c = ((quads_here + NT - 1) / NT) | 1;
  const int t0 = 4 * min(quads_here, tid * c), t1 = 4 * min(quads_here, tid * c + c);
  u64 sum = 0;
  unsigned count = 0;
  for (int j = 0; j < c; ++j) {
    const int i = min(t0 + 4 * j, t1);  // (past the thread's quads: one of the next, or the padding, left out)
    const float4 v = *reinterpret_cast<const float4*>(z + i);
    const float f[4] = {v.x, v.y, v.z, v.w};
    bool stay[4];
    cut.keeps4(f, i0 + i, stay);
    if (i >= t1) stay[0] = stay[1] = stay[2] = stay[3] = false;
    if (!__any_sync(0xffffffffu, stay[0] || stay[1] || stay[2] || stay[3])) continue;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const u64 w = W.biased(f[q]);
      if (stay[q]) {
        sum += w;
        ++count;
      }
    }
  }
  sum -= count * Weights::ONE;
  u64 total, kept;
  u64 before = block_scan<NT>(sum, S.sums, total);
  block_scan<NT>(count, S.sums, kept);
  R.publish(total, kept);
  total = kept = 0;
  for (int r = 0; r < CL; ++r) {
    if (r < rank) before += R.tot(r);
    total += R.tot(r);
    kept += R.tot2(r);
  }
  const double t = U * (double)total;
  const u64 goal = t > 0.0 ? min((u64)t, total - 1) : 0;
  if (goal < before || goal >= before + sum) return;
  for (int i = t0; i < t1; ++i) {
    if (!cut.keeps(z[i], i0 + i)) continue;
    before += W.fixed(z[i]);
    if (before > goal) {
      answer(i0 + i, (float)(W.scaled(z[i]) / (double)total), (int)kept);
      return;
    }
  }
}

size_t sample_bytes(int slice) { return sizeof(SampleShared) + ((size_t)slice + 8) * sizeof(float); }

}  // namespace

cudaError_t sample_init_device() {
  const int most = (int)sample_bytes(SM_SLICE);
  cudaError_t e = cudaFuncSetAttribute(sample_kernel<512>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(sample_kernel<1024>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
  return e;
}

cudaError_t dec_sample(const SampleArgs& a, int num_sms, cudaStream_t s) {
  int bits = 0;
  while ((1 << bits) < a.vocab) ++bits;
  // CTAs per row: as many as the slices ask for, more while every CTA has an SM to
  // itself (clusters of eight pack badly: half the SMs) and over two tokens a
  // thread.  Measured at 32 rows of 151,936 under top-p: 47.3 us for four, 49.6 for
  // eight; at 8 rows 45.9 and 30.5.  Where not even the least number fits so, eight
  // narrow CTAs, two per SM (64 rows without a filter: 44.7 us, four wide ones 46.8).
  int cl = 1;
  while (a.vocab > cl * SM_SLICE) cl *= 2;
  const auto fits = [&](int n) { return a.batch * n <= (n == 8 ? num_sms / 2 : num_sms); };
  if (!fits(cl) && cl > 1) cl = SM_MAX_CLUSTER;
  while (cl < SM_MAX_CLUSTER && a.vocab > cl * 1024 && fits(2 * cl)) cl *= 2;
  const int slice = ((a.vocab + cl - 1) / cl + 3) & ~3;  // whole quads
  // 1024 threads where a slice is long enough to hide in them and the SM is free
  const bool wide = fits(cl) && slice > 12288;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.batch * cl));
  cfg.blockDim = dim3(wide ? 1024 : 512);
  cfg.dynamicSmemBytes = sample_bytes(slice);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cl;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, wide ? sample_kernel<1024> : sample_kernel<512>, a, slice,
                            std::min(SM_FRAC, 62 - bits));
}

}  // namespace kq
