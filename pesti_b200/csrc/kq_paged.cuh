// kq_paged.cuh -- addressing of the paged key-value cache and the rotary
// angle, shared by the kernels of kq_paged.cu (host-callable, so that the
// index arithmetic can be checked without a GPU).
#pragma once

#include <stdint.h>

#include "kq_kernels.h"

namespace kq {

// Device error codes of the paged cache: input out of bounds (a word that no wait
// polls: other calls on the context go on as they are), and a wait that gave up.
enum : int { KV_ERR_PAGE = 51, KV_ERR_LEN = 52, KV_ERR_ROW = 53, KV_ERR_WAIT = 54 };

// A sequence's slots in use; where lens[b] is outside [0, most], *bad is set and the
// sequence counts as idle (held to `most`, a step would overwrite its last slot).
__host__ __device__ __forceinline__ int64_t kv_len(int32_t len, int64_t most, bool* bad) {
  *bad = len < 0 || len > most;
  return *bad ? 0 : (int64_t)len;
}

// Element offset of slot's row for one kv head, or -1 where the table's page
// is outside the pool.
__host__ __device__ __forceinline__ int64_t kv_row(const KvPool& p, int32_t page, int64_t slot, int head) {
  if (page < 0 || page >= p.pages) return -1;
  return (int64_t)page * p.page_ld + ((int64_t)head * p.page_size + slot % p.page_size) * p.hd;
}

// a * b * c past 2^60: scratch that no device holds, and whose size could wrap around.
inline bool kv_too_many(int64_t a, int64_t b, int64_t c) { return (double)a * (double)b * (double)c > 0x1p60; }

#ifdef __CUDACC__
__device__ __forceinline__ void kv_pdl_enter() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

__device__ __forceinline__ void kv_error(int* bad, int code) { atomicCAS(bad, 0, code); }

// Turns (of a full circle) per position of pair i: theta^(-i / half) / (2 pi).
__device__ __forceinline__ double rope_freq(int i, int half, double log2_theta) {
  return exp2(-(double)i / (double)half * log2_theta) * 0.15915494309189533577;
}
// cos / sin of pos * theta^(-i / half), in 64 bits: at position 100,000 an f32 angle
// is off by 4e-3.  To the nearest quarter turn, then the power series at |r| <= pi / 4,
// whose first terms left out are r^13 / 13! < 7e-12 and r^14 / 14! < 4e-13.
__device__ __forceinline__ void rope_turn(int32_t pos, double freq, double& c, double& s) {
  constexpr double F3 = 1.0 / 6, F5 = 1.0 / 120, F7 = 1.0 / 5040, F9 = 1.0 / 362880, F11 = 1.0 / 39916800;
  constexpr double F4 = 1.0 / 24, F6 = 1.0 / 720, F8 = 1.0 / 40320, F10 = 1.0 / 3628800, F12 = 1.0 / 479001600;
  const double t = 4.0 * ((double)pos * freq), n = rint(t);
  const double r = (t - n) * 1.5707963267948966192, x = -r * r;
  const double si = r * fma(x, fma(x, fma(x, fma(x, fma(x, F11, F9), F7), F5), F3), 1.0);
  const double co = fma(x, fma(x, fma(x, fma(x, fma(x, fma(x, F12, F10), F8), F6), F4), 0.5), 1.0);
  const int quarter = (int)(int64_t)n & 3;
  const double a = quarter & 1 ? si : co, b = quarter & 1 ? co : si;
  c = quarter == 1 || quarter == 2 ? -a : a;
  s = quarter & 2 ? -b : b;
}
// x c + y s to the nearest f32, c and s given as two f32 parts: the products' and the
// sum's roundings are worked out (a product's by fma, a sum's by Knuth's two-sum) and
// added last, 2^-46 of |x c| + |y s| is left.  Plain f32 sums would round another way
// to f16 at 2e-4 of the elements; FP64 takes more of the append kernel's 32 registers.
__device__ __forceinline__ float exact_dot2(float x, float c, float c_lo, float y, float s, float s_lo) {
  const float p = __fmul_rn(x, c), q = __fmul_rn(y, s), sum = __fadd_rn(p, q);
  const float z = __fsub_rn(sum, p), lost = __fadd_rn(__fsub_rn(p, __fsub_rn(sum, z)), __fsub_rn(q, z));
  const float pe = __fmaf_rn(x, c_lo, __fmaf_rn(x, c, -p)), qe = __fmaf_rn(y, s_lo, __fmaf_rn(y, s, -q));
  const float r = __fadd_rn(sum, __fadd_rn(lost, __fadd_rn(pe, qe)));
  return isfinite(sum) ? r : sum;
}
// A key's pair (x, y) turned.
__device__ __forceinline__ void turn_key(float x, float y, float c, float c_lo, float s, float s_lo, float& a,
                                         float& b) {
  a = exact_dot2(x, c, c_lo, -y, s, s_lo);
  b = exact_dot2(x, s, s_lo, y, c, c_lo);
}
#endif

}  // namespace kq
