// kq_sample.cu -- the next token of every sequence from its logits
// (include/pesti_decoder.h, kq_dec_sample): temperature, top-k, top-p, min-p and
// the draw from a given random number.
//
// Mathematics: in the order (logit descending, index ascending) each filter
// keeps a prefix, so every one is a threshold on the 64-bit word (key of the
// logit, ~index).  The weights 2^((z - max) log2 e / T) are 64-bit fixed point,
// 2^44 or less for the largest: their sums are exact whatever their order, and a
// draw next to the border of two tokens falls on the same side on every run.
//
// What bounds it: one read of the logits from HBM, and where the weights of the
// whole vocabulary are summed about 12 FP64 instructions each.  A cluster of up
// to eight CTAs shares a row: every CTA keeps its slice of the logits in shared
// memory, so they are read once, and the slices' histograms are joined over
// distributed shared memory.
//  * top-k: counts in 2048 bins of the distance from the maximum; the few
//    candidates down to the bin of the k-th go to one CTA, which ranks them
//    against one another and applies the other filters to them;
//  * top-p over more than that: weights in the same bins, then the bin of the
//    border: its tokens are ranked by one CTA where they are few, else the bins
//    are refined over the words themselves (at most 64 bits, 11 at a time);
//  * the draw: sums per thread over consecutive tokens, and one thread walks the
//    stretch that holds it.
#include "kq_common.cuh"
#include "kq_kernels.h"

#include <cooperative_groups.h>
#include <float.h>
#include <math.h>

namespace kq {
namespace {

namespace cg = cooperative_groups;
typedef unsigned long long u64;

constexpr int SM_THREADS = 512, SM_WARPS = SM_THREADS / 32;
constexpr int SM_BINS = 2048;
constexpr int SM_LIST = 1024;     // candidates one CTA ranks
constexpr int SM_MAX_CLUSTER = 8;
constexpr int SM_SLICE = SAMPLE_MAX_VOCAB / SM_MAX_CLUSTER;  // logits a CTA can hold
constexpr int SM_FRAC = 44;       // weights below 2^-45 (distances above 31.2 T) count as zero

// f32 -> unsigned with the same order
__device__ __forceinline__ uint32_t order_key(float f) {
  const uint32_t u = __float_as_uint(f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_logit(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
// a token's word: greater is earlier in the order
__device__ __forceinline__ u64 word_of(float z, int i) { return (u64)order_key(z) << 32 | (uint32_t)~i; }

struct SampleShared {
  double pow2[64];             // 2^(i / 64)
  u64 sums[SM_WARPS];
  u64 tot[SM_MAX_CLUSTER];     // per CTA of the cluster, written by each
  u64 tot2[SM_MAX_CLUSTER];
  u64 res[3];                  // what one CTA found for all
  unsigned listed;             // first CTA: candidates so far
  uint32_t lo[SM_BINS], hi[SM_BINS];  // histogram, 64-bit sums as two words
  u64 list[SM_LIST], weight[SM_LIST];  // first CTA: candidates
};

__device__ __forceinline__ u64 warp_sum(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Exclusive sum over the block; `total` gets the sum.
__device__ __forceinline__ u64 block_scan(u64 v, u64* sums, u64& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  u64 x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) sums[warp] = x;
  __syncthreads();
  u64 before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < SM_WARPS; ++w) {
    if (w < warp) before += sums[w];
    total += sums[w];
  }
  return before + x - v;
}

// The weights of one row.
struct Weights {
  double c, scale, zmax;  // 64 log2 e / T, 2^frac, the greatest logit
  const double* pow2;
  // 2^(frac + (z - max) log2 e / T) to about 1e-13; 0 where it is below 1/2.
  // 2^t = 2^n/64 2^r with |r| <= 1/128: a table and the exponential series in r.
  __device__ __forceinline__ double scaled(float z) const {
    const double t = ((double)z - zmax) * c;
    if (t < -64.0 * 46.0) return 0.0;
    constexpr double ROUND = 6755399441055744.0;  // 1.5 2^52: the sum's last bits are the nearest integer
    const double nd = t + ROUND;
    const int n = __double2loint(nd);
    const double r = t - (nd - ROUND);
    constexpr double A = 0.010830424696249145;  // ln 2 / 64
    const double p = fma(r, fma(r, fma(r, fma(r, A * A * A * A / 24, A * A * A / 6), A * A / 2), A), 1.0);
    const double e = __hiloint2double((1023 + (n >> 6)) << 20, 0);
    return pow2[n & 63] * p * e * scale;
  }
  __device__ __forceinline__ u64 fixed(float z) const {
    return (u64)__double_as_longlong(scaled(z) + 4503599627370496.0) & 0xfffffffffffffull;  // + 2^52: rounded
  }
};

// One row's CTAs: their slice and what they share.
struct Row {
  cg::cluster_group cluster;
  SampleShared& S;
  float* z;
  int CL, rank, i0, n;

  // Two values per CTA, known to every CTA after the next cluster.sync().
  __device__ __forceinline__ void publish(u64 a, u64 b) {
    if (threadIdx.x < CL) {
      SampleShared* to = cluster.map_shared_rank(&S, threadIdx.x);
      to->tot[rank] = a;
      to->tot2[rank] = b;
    }
  }
  __device__ __forceinline__ void publish_res(int k, u64 v) {
    for (int r = 0; r < CL; ++r) cluster.map_shared_rank(&S, r)->res[k] = v;
  }

  // Histogram of measure(z) over bin_of(z, word) (-1: left out) of all slices; the
  // bin in which the running sum from bin 0 reaches target(total).  False where
  // it does not.  `left`: how much of the bin it takes; `upto`: the sum with the bin.
  template <class Bin, class Measure, class Target>
  __device__ bool find_bin(Bin bin_of, Measure measure, Target target_of, int& bin, u64& left, u64& upto) {
    for (int e = threadIdx.x; e < SM_BINS; e += SM_THREADS) S.lo[e] = S.hi[e] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += SM_THREADS) {
      const int k = bin_of(z[i], word_of(z[i], i0 + i));
      if (k < 0) continue;
      const u64 m = measure(z[i]);
      const uint32_t l = (uint32_t)m;
      const uint32_t old = atomicAdd(&S.lo[k], l);
      const uint32_t h = (uint32_t)(m >> 32) + (old + l < old);  // the carry
      if (h) atomicAdd(&S.hi[k], h);
    }
    cluster.sync();
    const int bins = SM_BINS / CL, per = (bins + SM_THREADS - 1) / SM_THREADS;  // this CTA joins bins [rank bins, ..)
    constexpr int MOST = SM_BINS / SM_THREADS;
    u64 m[MOST], sum = 0;
#pragma unroll
    for (int q = 0; q < MOST; ++q) {
      m[q] = 0;
      const int e = threadIdx.x * per + q;
      if (q < per && e < bins)
        for (int r = 0; r < CL; ++r) {
          const SampleShared* from = cluster.map_shared_rank(&S, r);
          m[q] += (u64)from->hi[rank * bins + e] << 32 | from->lo[rank * bins + e];
        }
      sum += m[q];
    }
    u64 total;
    u64 before = block_scan(sum, S.sums, total);
    publish(total, 0);
    cluster.sync();
    u64 all = 0;
    for (int r = 0; r < CL; ++r) {
      if (r < rank) before += S.tot[r];
      all += S.tot[r];
    }
    const u64 target = target_of(all);
    if (target > all) return false;
#pragma unroll
    for (int q = 0; q < MOST; ++q) {
      if (target > before && target <= before + m[q]) {
        publish_res(0, (u64)(rank * bins + threadIdx.x * per + q));
        publish_res(1, target - before);
        publish_res(2, before + m[q]);
      }
      before += m[q];
    }
    cluster.sync();
    bin = (int)S.res[0];
    left = S.res[1];
    upto = S.res[2];
    return true;
  }

  // The tokens of pred(z, word) to the first CTA's list, counted there (what does
  // not fit is dropped).  After the call another CTA may look at the first one's
  // memory only where a cluster.sync() follows.
  template <class Pred>
  __device__ void gather(Pred pred) {
    SampleShared* first = cluster.map_shared_rank(&S, 0);
    for (int i = threadIdx.x; i < n; i += SM_THREADS) {
      const u64 w = word_of(z[i], i0 + i);
      if (!pred(z[i], w)) continue;
      const unsigned at = atomicAdd(&first->listed, 1u);
      if (at < SM_LIST) first->list[at] = w;
    }
    cluster.sync();
  }

  // The word of the token at which the running sum of measure(z), over the tokens
  // of pred from the greatest word, reaches `left` (their sum is at least that).
  template <class Measure, class Pred>
  __device__ u64 border(Measure measure, u64 left, Pred pred) {
    gather(pred);
    const unsigned listed = *cluster.map_shared_rank(&S.listed, 0);
    if (listed <= SM_LIST) {
      if (rank == 0) {
        for (unsigned e = threadIdx.x; e < listed; e += SM_THREADS) S.weight[e] = measure(key_logit((uint32_t)(S.list[e] >> 32)));
        __syncthreads();
        for (unsigned e = threadIdx.x; e < listed; e += SM_THREADS) {
          const u64 w = S.list[e];
          u64 before = 0;
          for (unsigned j = 0; j < listed; ++j) before += S.list[j] > w ? S.weight[j] : 0;
          if (before < left && left <= before + S.weight[e]) publish_res(0, w);
        }
      }
      cluster.sync();
      if (rank == 0 && threadIdx.x == 0) S.listed = 0;
      return S.res[0];
    }
    // too many: refine over the words, from their exact range
    u64 low = ~0ull, high = 0;
    for (int i = threadIdx.x; i < n; i += SM_THREADS) {
      const u64 w = word_of(z[i], i0 + i);
      if (!pred(z[i], w)) continue;
      low = w < low ? w : low;
      high = w > high ? w : high;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const u64 a = __shfl_xor_sync(0xffffffffu, low, o), c = __shfl_xor_sync(0xffffffffu, high, o);
      low = a < low ? a : low;
      high = c > high ? c : high;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) {
      S.list[threadIdx.x >> 5] = low;
      S.weight[threadIdx.x >> 5] = high;
    }
    __syncthreads();
    for (int w = 0; w < SM_WARPS; ++w) {
      low = S.list[w] < low ? S.list[w] : low;
      high = S.weight[w] > high ? S.weight[w] : high;
    }
    publish(low, high);
    cluster.sync();
    if (rank == 0 && threadIdx.x == 0) S.listed = 0;
    for (int r = 0; r < CL; ++r) {
      low = S.tot[r] < low ? S.tot[r] : low;
      high = S.tot2[r] > high ? S.tot2[r] : high;
    }
    while (low < high) {
      const int shift = max(0, 64 - __clzll((long long)(high - low)) - 11);
      int bin = 0;
      u64 upto;
      const u64 goal = left;
      find_bin([&](float f, u64 w) { return w >= low && w <= high && pred(f, w) ? SM_BINS - 1 - (int)((w - low) >> shift) : -1; },
               measure, [&](u64) { return goal; }, bin, left, upto);
      low += (u64)(SM_BINS - 1 - bin) << shift;
      const u64 top = low + ((1ull << shift) - 1);
      high = top < high ? top : high;
    }
    return low;
  }
};

__global__ void __launch_bounds__(SM_THREADS, 2) sample_kernel(const SampleArgs A, int slice, int frac) {
  extern __shared__ __align__(16) uint8_t dyn[];
  SampleShared& S = *reinterpret_cast<SampleShared*>(dyn);
  cg::cluster_group cluster = cg::this_cluster();
  const int CL = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int64_t b = blockIdx.x / CL;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int i0 = min(A.vocab, rank * slice), n = min(A.vocab, i0 + slice) - i0;  // this CTA's tokens
  float* z = reinterpret_cast<float*>(dyn + sizeof(SampleShared));
  Row R{cluster, S, z, CL, rank, i0, n};
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (tid < 64) S.pow2[tid] = exp2((double)tid / 64.0);
  if (tid == 0) S.listed = 0;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const float T = A.temperature ? A.temperature[b] : 1.f;
  int K = A.top_k ? A.top_k[b] : 0;
  const double P = A.top_p ? (double)A.top_p[b] : 1.0, M = A.min_p ? (double)A.min_p[b] : 0.0;
  const double U = (double)A.u[b];

  // ---- the slice into shared memory; the greatest word, and how many tokens can be drawn ----
  const float* row = A.logits + b * A.ld + i0;
  u64 best = 0, able = 0;
#pragma unroll 8
  for (int i = tid; i < n; i += SM_THREADS) {
    float f = row[i] + 0.f;  // -0 as 0
    if (isnan(f)) f = -INFINITY;
    z[i] = f;
    const u64 w = word_of(f, i0 + i);
    best = w > best ? w : best;
    able += f > -INFINITY;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const u64 y = __shfl_xor_sync(0xffffffffu, best, o);
    best = y > best ? y : best;
  }
  able = warp_sum(able);
  if (lane == 0) {
    S.list[warp] = best;
    S.weight[warp] = able;
  }
  cluster.sync();  // every CTA has started: its shared memory may be written
  best = able = 0;
  for (int w = 0; w < SM_WARPS; ++w) {
    best = S.list[w] > best ? S.list[w] : best;
    able += S.weight[w];
  }
  R.publish(best, able);
  cluster.sync();
  best = able = 0;
  for (int r = 0; r < CL; ++r) {
    best = S.tot[r] > best ? S.tot[r] : best;
    able += S.tot2[r];
  }
  auto answer = [&](int token, float prob, int kept) {
    A.tokens[b] = token;
    if (A.prob) A.prob[b] = prob;
    if (A.kept) A.kept[b] = kept;
  };
  if (able == 0) {  // no token is possible
    if (rank == 0 && tid == 0) answer(-1, 0.f, 0);
    return;
  }
  if (!(T > 0.f) || K == 1 || !(P > 0.0) || !(M <= 1.0)) {
    if (rank == 0 && tid == 0) answer((int)~(uint32_t)best, 1.f, 1);
    return;
  }
  float zmax = key_logit((uint32_t)(best >> 32));
  if (isinf(zmax)) {  // only tokens of +inf carry weight: 0 for them, the least number for the others
    for (int i = tid; i < n; i += SM_THREADS)
      z[i] = z[i] == INFINITY ? 0.f : z[i] > -INFINITY ? -FLT_MAX : -INFINITY;
    zmax = 0.f;
    best = (u64)order_key(0.f) << 32 | (uint32_t)best;
    __syncthreads();
  }
  Weights W;
  W.c = 92.332482616893656 / (double)T;  // 64 log2 e
  W.scale = (double)(1ull << frac);
  W.zmax = (double)zmax;
  W.pow2 = S.pow2;
  auto fixed = [&](float f) { return W.fixed(f); };
  auto one = [](float) { return 1ull; };

  u64 thr = (u64)(order_key(-INFINITY) + 1) << 32;  // the least word that stays
  if (K > 0 && (u64)K < able) {
    // counts of the distance from the maximum, 64 bins per unit
    auto near = [&](float f) {
      const float q = (zmax - f) * 64.f;
      return q < (float)SM_BINS ? (int)q : -1;
    };
    int bin = 0;
    u64 left = (u64)K, upto = 0;
    const bool found = R.find_bin([&](float f, u64) { return near(f); }, one, [&](u64) { return (u64)K; }, bin, left, upto);
    if (found && upto <= SM_LIST) {
      R.gather([&](float f, u64) {
        const int k = near(f);
        return k >= 0 && k <= bin;
      });
      if (rank != 0) return;
      const int m = (int)upto;
      // ---- one CTA has the candidates: all filters and the draw by comparing them with one another ----
      constexpr int PER = SM_LIST / SM_THREADS;
      u64 mine[PER], w[PER], total = 0;
      int place[PER];
#pragma unroll
      for (int q = 0; q < PER; ++q) {
        const int e = tid + q * SM_THREADS;
        mine[q] = e < m ? S.list[e] : 0;
        w[q] = 0;
        place[q] = 0;
        if (e < m) {
          for (int j = 0; j < m; ++j) place[q] += S.list[j] > mine[q];
          if (place[q] < K) w[q] = W.fixed(key_logit((uint32_t)(mine[q] >> 32)));
          S.weight[e] = w[q];
        }
        total += w[q];
      }
      block_scan(total, S.sums, total);
      const double goal_p = ceil(P * (double)total);
      u64 kept = 0, sum = 0;
#pragma unroll
      for (int q = 0; q < PER; ++q) {
        const int e = tid + q * SM_THREADS;
        bool stay = e < m && place[q] < K;
        if (stay && place[q] > 0) {
          if (P < 1.0) {
            u64 before = 0;
            for (int j = 0; j < m; ++j) before += S.list[j] > mine[q] ? S.weight[j] : 0;
            stay = (double)before < goal_p;
          }
          stay = stay && W.scaled(key_logit((uint32_t)(mine[q] >> 32))) >= M * W.scale;
        }
        if (!stay) w[q] = 0;
        kept += stay;
        sum += w[q];
      }
      block_scan(kept, S.sums, kept);
      block_scan(sum, S.sums, total);  // (its barriers end the reads of S.weight)
#pragma unroll
      for (int q = 0; q < PER; ++q)
        if (tid + q * SM_THREADS < m) S.weight[tid + q * SM_THREADS] = w[q];
      __syncthreads();
      const double t = U * (double)total;
      const u64 goal = t > 0.0 ? min((u64)t, total - 1) : 0;
#pragma unroll
      for (int q = 0; q < PER; ++q) {
        if (w[q] == 0) continue;
        u64 before = 0;  // a lower index has a greater low half of the word
        for (int j = 0; j < m; ++j) before += (uint32_t)S.list[j] > (uint32_t)mine[q] ? S.weight[j] : 0;
        if (before <= goal && goal < before + w[q])
          answer((int)~(uint32_t)mine[q], (float)(W.scaled(key_logit((uint32_t)(mine[q] >> 32))) / (double)total),
                 (int)kept);
      }
      return;
    }
    const u64 floor = thr;
    thr = found ? R.border(one, left, [&](float f, u64) { return near(f) == bin; })
                : R.border(one, (u64)K, [&](float, u64 w) { return w >= floor; });
  }
  if (P < 1.0) {
    const float per_t = 64.f / T;
    auto near = [&](float f) {
      const float d = zmax - f, q = d * per_t;
      return d > 0.f ? (q < (float)SM_BINS ? (int)q : -1) : 0;  // beyond: weight 0
    };
    int bin = 0;
    u64 left = 0, upto;
    const u64 floor = thr;
    R.find_bin([&](float f, u64 w) { return w >= floor ? near(f) : -1; }, fixed,
               [&](u64 all) { return min(max((u64)ceil(P * (double)all), 1ull), all); }, bin, left, upto);
    thr = R.border(fixed, left, [&](float f, u64 w) { return w >= floor && near(f) == bin; });
  }

  // ---- the draw: thread t sums tokens [t c, (t + 1) c) of the slice (c odd: no bank is hit twice) ----
  const int c = ((n + SM_THREADS - 1) / SM_THREADS) | 1;
  const int t0 = min(n, tid * c), t1 = min(n, t0 + c);
  const double least = M * W.scale;
  u64 sum = 0, count = 0;
  for (int i = t0; i < t1; ++i) {
    const u64 w = word_of(z[i], i0 + i);
    if (w < thr) continue;
    const double s = W.scaled(z[i]);
    if (!(s >= least) && w != best) continue;
    sum += (u64)__double_as_longlong(s + 4503599627370496.0) & 0xfffffffffffffull;
    ++count;
  }
  u64 total, kept;
  u64 before = block_scan(sum, S.sums, total);
  block_scan(count, S.sums, kept);
  __syncthreads();
  R.publish(total, kept);
  cluster.sync();
  total = kept = 0;
  for (int r = 0; r < CL; ++r) {
    if (r < rank) before += S.tot[r];
    total += S.tot[r];
    kept += S.tot2[r];
  }
  const double t = U * (double)total;
  const u64 goal = t > 0.0 ? min((u64)t, total - 1) : 0;
  if (goal < before || goal >= before + sum) return;
  for (int i = t0; i < t1; ++i) {
    const u64 w = word_of(z[i], i0 + i);
    if (w < thr) continue;
    const double s = W.scaled(z[i]);
    if (!(s >= least) && w != best) continue;
    before += (u64)__double_as_longlong(s + 4503599627370496.0) & 0xfffffffffffffull;
    if (before > goal) {
      answer(i0 + i, (float)(s / (double)total), (int)kept);
      return;
    }
  }
}

size_t sample_smem(int slice) { return sizeof(SampleShared) + (size_t)slice * sizeof(float); }

}  // namespace

cudaError_t sample_init_device() {
  return cudaFuncSetAttribute(sample_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sample_smem(SM_SLICE));
}

cudaError_t dec_sample(const SampleArgs& a, cudaStream_t s) {
  int bits = 0;
  while ((1 << bits) < a.vocab) ++bits;
  // as many CTAs per row as the slices ask for, and more while a slice has over
  // two tokens a thread
  int cl = 1;
  while (cl < SM_MAX_CLUSTER && (a.vocab > cl * SM_SLICE || a.vocab > cl * 2 * SM_THREADS)) cl *= 2;
  const int slice = (a.vocab + cl - 1) / cl;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.batch * cl));
  cfg.blockDim = dim3(SM_THREADS);
  cfg.dynamicSmemBytes = sample_smem(slice);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cl;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, sample_kernel, a, slice, std::min(SM_FRAC, 62 - bits));
}

}  // namespace kq
