// kq_sample.cu -- the next token of every sequence from its logits
// (include/pesti_decoder.h, kq_dec_sample): temperature, top-k, top-p, min-p and
// the draw from a given random number, one CTA per sequence.
//
// In the order (logit descending, index ascending) each filter keeps a prefix,
// so all of them together are one threshold: a key, and how many of the tokens
// with that key stay (the lowest indices).  The weights e^((z - max) / T) are
// held as 64-bit fixed point (2^F for the largest, F such that the vocabulary's
// sum fits): sums are exact and do not depend on their order, so a draw next to
// a border between two tokens falls on the same side on every run.
#include "kq_common.cuh"
#include "kq_kernels.h"

#include <math.h>

#include <algorithm>

namespace kq {
namespace {

typedef unsigned long long u64;

__device__ __forceinline__ void pdl_enter() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

__device__ __forceinline__ uint32_t order_key(float f) {
  const uint32_t u = __float_as_uint(isnan(f) ? -INFINITY : f + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
constexpr uint32_t KEY_NONE = 0x007fffffu;  // the key of -inf
__device__ __forceinline__ float key_logit(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

constexpr int SM_THREADS = 1024;

__global__ void __launch_bounds__(SM_THREADS) sample_kernel(const SampleArgs A, int frac) {
  pdl_enter();
  __shared__ u64 hist[256];
  __shared__ u64 red[SM_THREADS];
  __shared__ u64 pick[3];
  const int64_t b = blockIdx.x;
  const int tid = threadIdx.x, V = A.vocab;
  const float* z = A.logits + b * A.ld;
  // the greatest key and its first index, as one word
  u64 best = 0;
  for (int i = tid; i < V; i += SM_THREADS) {
    const u64 w = (u64)order_key(z[i]) << 32 | (uint32_t)~i;
    best = w > best ? w : best;
  }
  red[tid] = best;
  __syncthreads();
  for (int o = SM_THREADS / 2; o > 0; o >>= 1) {
    if (tid < o) red[tid] = red[tid + o] > red[tid] ? red[tid + o] : red[tid];
    __syncthreads();
  }
  const uint32_t kmax = (uint32_t)(red[0] >> 32);
  const int first = (int)~(uint32_t)red[0];
  __syncthreads();
  auto answer = [&](int token, float prob, int kept) {
    A.tokens[b] = token;
    if (A.prob) A.prob[b] = prob;
    if (A.kept) A.kept[b] = kept;
  };
  if (kmax <= KEY_NONE) {  // no token is possible
    if (tid == 0) answer(-1, 0.f, 0);
    return;
  }
  const float T = A.temperature ? A.temperature[b] : 1.f;
  const int K = A.top_k ? A.top_k[b] : 0;
  const double P = A.top_p ? (double)A.top_p[b] : 1.0, M = A.min_p ? (double)A.min_p[b] : 0.0;
  if (!(T > 0.f) || K == 1 || !(P > 0.0) || !(M <= 1.0)) {
    if (tid == 0) answer(first, 1.f, 1);
    return;
  }
  const double zmax = (double)key_logit(kmax);
  auto weight = [&](uint32_t k) {  // e^((z - max) / T)
    return k == kmax ? 1.0 : exp(((double)key_logit(k) - zmax) / (double)T);
  };
  auto fixed = [&](double w) { return (u64)(w * (double)(1ull << frac) + 0.5); };
  // Walk the digits of the key from the top: after them, the key at which the
  // running sum (tokens or weight) from above reaches `left`.
  uint32_t thr = KEY_NONE;
  u64 quota = 0;  // tokens of key thr that stay
  auto select = [&](bool by_weight, u64 left, uint32_t floor_key, u64 floor_quota, u64& at) {
    uint32_t prefix = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int e = tid; e < 256; e += SM_THREADS) hist[e] = 0;
      __syncthreads();
      for (int i = tid; i < V; i += SM_THREADS) {
        const uint32_t k = order_key(z[i]);
        if (k <= floor_key || (shift < 24 && (k >> (shift + 8)) != prefix)) continue;
        atomicAdd(&hist[(k >> shift) & 255u], by_weight ? fixed(weight(k)) : 1ull);
      }
      if (tid == 0 && floor_quota && (shift == 24 || (floor_key >> (shift + 8)) == prefix))
        atomicAdd(&hist[(floor_key >> shift) & 255u], floor_quota * (by_weight ? fixed(weight(floor_key)) : 1ull));
      __syncthreads();
      if (tid == 0) {
        int d = 255;
        while (d > 0 && hist[d] < left) left -= hist[d--];
        pick[0] = d;
        pick[1] = left;
      }
      __syncthreads();
      prefix = prefix << 8 | (uint32_t)pick[0];
      left = pick[1];
      __syncthreads();
    }
    at = left;
    return prefix;
  };
  auto block_sum = [&](u64 v) {
    red[tid] = v;
    __syncthreads();
    for (int o = SM_THREADS / 2; o > 0; o >>= 1) {
      if (tid < o) red[tid] += red[tid + o];
      __syncthreads();
    }
    const u64 r = red[0];
    __syncthreads();
    return r;
  };
  if (K > 0) {
    u64 n = 0;
    for (int i = tid; i < V; i += SM_THREADS) n += order_key(z[i]) > KEY_NONE;
    if (block_sum(n) > (u64)K) thr = select(false, (u64)K, KEY_NONE, 0, quota);
  }
  if (P < 1.0) {
    u64 s = 0;
    for (int i = tid; i < V; i += SM_THREADS) {
      const uint32_t k = order_key(z[i]);
      if (k > thr) s += fixed(weight(k));
    }
    if (tid == 0 && quota) s += quota * fixed(weight(thr));
    s = block_sum(s);
    const u64 target = max(1ull, (u64)ceil(P * (double)s));
    u64 left;
    thr = select(true, min(target, s), thr, quota, left);
    const u64 w = fixed(weight(thr));
    quota = (left + w - 1) / w;
  }
  // thread t owns tokens [t c, (t + 1) c): ties are ranked and the draw is found in index order
  const int c = (V + SM_THREADS - 1) / SM_THREADS, i0 = min(V, tid * c), i1 = min(V, i0 + c);
  u64 ties = 0;
  for (int i = i0; i < i1; ++i) ties += order_key(z[i]) == thr;
  red[tid] = ties;
  __syncthreads();
  u64 rank0 = 0;
  for (int t = 0; t < tid; ++t) rank0 += red[t];
  __syncthreads();
  u64 sum = 0, n = 0;
  auto visit = [&](auto f) {
    u64 rank = rank0;
    for (int i = i0; i < i1; ++i) {
      const uint32_t k = order_key(z[i]);
      if (k < thr || (k == thr && rank++ >= quota)) continue;
      const double w = weight(k);
      if (w < M) continue;
      f(i, w);
    }
  };
  visit([&](int, double w) {
    sum += fixed(w);
    ++n;
  });
  const u64 kept = block_sum(n);
  red[tid] = sum;
  __syncthreads();
  u64 before = 0, total = 0;
  for (int t = 0; t < SM_THREADS; ++t) {
    if (t == tid) before = total;
    total += red[t];
  }
  const double t = (double)A.u[b] * (double)total;
  const u64 goal = t > 0.0 ? min((u64)t, total - 1) : 0;
  if (before <= goal && goal < before + sum) {
    bool found = false;
    visit([&](int i, double w) {
      before += fixed(w);
      if (!found && before > goal) {
        found = true;
        answer(i, (float)(w / ((double)total / (double)(1ull << frac))), (int)kept);
      }
    });
  }
}

}  // namespace

cudaError_t sample_init_device() { return cudaSuccess; }

cudaError_t dec_sample(const SampleArgs& a, cudaStream_t s) {
  int bits = 0;
  while ((1 << bits) < a.vocab) ++bits;
  return launch_pdl(sample_kernel, dim3((unsigned)a.batch), dim3(SM_THREADS), 0, s, a, 62 - bits);
}

}  // namespace kq
