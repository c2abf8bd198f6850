// kq_paged.cu -- a paged f16 key-value cache: appending rows and eviction by
// accumulated attention weight (include/pesti_decoder.h, kq_kv_append and
// kq_kv_evict).
#include "kq_paged.cuh"

#include <cuda_fp16.h>
#include <math.h>

#include <algorithm>

namespace kq {
namespace {

// ---- append ---------------------------------------------------------------------
// One CTA per row: the row's angles once (in 64 bits, hd / 2 of them) into shared
// memory, then four consecutive pairs of a head per thread and step, AP_STEPS
// steps' loads in flight.  Bound by the row's bytes: f32 in, f32 q and f16 k, v out.
constexpr int AP_THREADS = 256, AP_STEPS = 4, AP_MAX_HALF = 128;

// Four floats at p, in one access where `vec` (p is then 16-byte aligned).
__device__ __forceinline__ float4 load4(const float* p, bool vec) {
  return vec ? *reinterpret_cast<const float4*>(p) : make_float4(p[0], p[1], p[2], p[3]);
}
__device__ __forceinline__ void store4(float* p, float4 v, bool vec) {
  if (vec) {
    *reinterpret_cast<float4*>(p) = v;
  } else {
    p[0] = v.x;
    p[1] = v.y;
    p[2] = v.z;
    p[3] = v.w;
  }
}
__device__ __forceinline__ uint2 halves(float4 v) {
  const __half2 a = __floats2half2_rn(v.x, v.y), b = __floats2half2_rn(v.z, v.w);
  return make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

__global__ void __launch_bounds__(AP_THREADS) kv_append_kernel(const KvAppendArgs A, bool vec_in, bool vec_out) {
  kv_pdl_enter();
  __shared__ float4 turn_c[AP_MAX_HALF / 4], turn_s[AP_MAX_HALF / 4];
  const int hd = A.pool.hd, half = hd / 2, hkv = A.pool.hkv, tid = threadIdx.x;
  const int64_t r = blockIdx.x;
  const int32_t slot = A.slots[r];
  if (slot < 0) return;
  const int64_t b = A.seqs ? A.seqs[r] : r;
  if (b < 0 || b >= A.batch || slot >= A.table_ld * A.pool.page_size || (A.slot_pos && slot >= A.track_ld)) {
    if (tid == 0) kv_error(A.err, KV_ERR_ROW);
    return;
  }
  const int32_t page = A.table[b * A.table_ld + slot / A.pool.page_size];
  const int32_t pos = A.pos ? A.pos[r] : slot;
  if (tid < half)
    rope_turn(pos, tid, half, A.log2_theta, reinterpret_cast<float*>(turn_c)[tid], reinterpret_cast<float*>(turn_s)[tid]);
  const int64_t row0 = kv_row(A.pool, page, slot, 0), head_ld = (int64_t)A.pool.page_size * hd;
  if (row0 < 0 && tid == 0) kv_error(A.err, KV_ERR_PAGE);
  __syncthreads();
  const float* row = A.qkv + r * A.ld;
  float* q_out = A.q_out ? A.q_out + r * A.q_ld : nullptr;
  __half* kc = static_cast<__half*>(A.pool.k) + row0;
  __half* vc = static_cast<__half*>(A.pool.v) + row0;
  // q and k heads (q only where it is wanted)
  const int quads = half / 4, first = q_out ? 0 : A.hq * quads, end = (A.hq + hkv) * quads;
  for (int e0 = first + tid; e0 < end; e0 += AP_STEPS * AP_THREADS) {
    float4 x[AP_STEPS], y[AP_STEPS];
#pragma unroll
    for (int k = 0; k < AP_STEPS; ++k) {
      const int e = e0 + k * AP_THREADS;
      if (e >= end) break;
      const float* p = row + (int64_t)(e / quads) * hd + 4 * (e % quads);
      x[k] = load4(p, vec_in);
      y[k] = load4(p + half, vec_in);
    }
#pragma unroll
    for (int k = 0; k < AP_STEPS; ++k) {
      const int e = e0 + k * AP_THREADS;
      if (e >= end) break;
      const int head = e / quads, i = 4 * (e % quads);
      const float4 c = turn_c[i / 4], s = turn_s[i / 4];
      const float4 a = make_float4(x[k].x * c.x - y[k].x * s.x, x[k].y * c.y - y[k].y * s.y,
                                   x[k].z * c.z - y[k].z * s.z, x[k].w * c.w - y[k].w * s.w);
      const float4 d = make_float4(x[k].x * s.x + y[k].x * c.x, x[k].y * s.y + y[k].y * c.y,
                                   x[k].z * s.z + y[k].z * c.z, x[k].w * s.w + y[k].w * c.w);
      if (head < A.hq) {
        float* o = q_out + (int64_t)head * hd + i;
        store4(o, a, vec_out);
        store4(o + half, d, vec_out);
      } else if (row0 >= 0) {
        __half* o = kc + (head - A.hq) * head_ld + i;
        *reinterpret_cast<uint2*>(o) = halves(a);
        *reinterpret_cast<uint2*>(o + half) = halves(d);
      }
    }
  }
  if (row0 < 0) return;
  for (int e = tid; e < hkv * (hd / 4); e += AP_THREADS) {
    const int h = e / (hd / 4), i = 4 * (e - h * (hd / 4));
    *reinterpret_cast<uint2*>(vc + h * head_ld + i) = halves(load4(row + (int64_t)(A.hq + hkv + h) * hd + i, vec_in));
  }
  if (A.slot_pos)
    for (int h = tid; h < hkv; h += AP_THREADS) A.slot_pos[(b * hkv + h) * A.track_ld + slot] = pos;
}

// ---- eviction ---------------------------------------------------------------------
// Kept are the `keep` slots that come first in the order (protected slots, then
// by mass descending, ties by slot).  Attention does not depend on the order of
// the slots, so only the holes below `keep` are filled, in ascending order, with
// the kept slots above it: the fewest rows move, and no row that is read is
// written.
//
// One CTA selects for a (sequence, kv head): the key of the last slot kept by
// three passes over 11-bit digits, then the lists of holes and kept slots above
// by sums over the threads, each owning consecutive slots.  Keys are read from
// global memory once and stay in shared memory (up to EV_PIECE slots; longer
// caches go piece by piece).  A second kernel moves the rows: it is bound by
// them, the first by the latency of its passes.
constexpr int EV_THREADS = 1024, EV_BINS = 2048, EV_PIECE = 40960;
constexpr size_t EV_SMEM = (size_t)EV_PIECE * 4;

// f32 -> unsigned with the same order; -0 as 0, NaN as -inf
__device__ __forceinline__ uint32_t order_key(float f) {
  const uint32_t u = __float_as_uint(isnan(f) ? -INFINITY : f + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Exclusive sum over the block (a multiple of 32 threads); `total` gets the sum.
__device__ __forceinline__ int block_scan(int v, int* warp_sums, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  int before = 0;
  total = 0;
  for (int w = 0; w < warps; ++w) {
    if (w < warp) before += warp_sums[w];
    total += warp_sums[w];
  }
  return before + x - v;
}

struct EvictPlan {  // one (sequence, kv head)
  int moves, new_len;
  int pad[2];
};

// Per (sequence, kv head) after the plans: the holes, then as many movers (holes
// lie below `keep`, movers above it: together at most track_ld).
__host__ __device__ __forceinline__ int64_t evict_list(int64_t track_ld) { return (track_ld + 3) & ~int64_t(3); }

__global__ void __launch_bounds__(EV_THREADS) kv_evict_select_kernel(const KvEvictArgs A) {
  extern __shared__ uint32_t keys[];
  __shared__ unsigned hist[EV_BINS];
  __shared__ int sums[32];
  __shared__ int pick[3];  // digit, how many of it are kept, how many there are
  const int hk = blockIdx.x, hkv = A.pool.hkv, tid = threadIdx.x;
  const int64_t b = blockIdx.y, bh = b * hkv + hk;
  for (int e = tid; e < EV_BINS; e += EV_THREADS) hist[e] = 0;
  __syncthreads();
  kv_pdl_enter();
  bool bad;
  const int len = (int)kv_len(A.lens[b], min(A.table_ld * A.pool.page_size, A.track_ld), &bad);
  if (bad && tid == 0) kv_error(A.err, KV_ERR_LEN);
  const int keep = A.keep, new_len = min(len, keep);
  EvictPlan* plan = static_cast<EvictPlan*>(A.scratch) + bh;
  int* list = reinterpret_cast<int*>(static_cast<EvictPlan*>(A.scratch) + A.batch * hkv) + bh * evict_list(A.track_ld);
  const float* mass = A.mass + bh * A.track_ld;
  const int32_t* spos = A.slot_pos + bh * A.track_ld;
  float* mass_out = A.mass_out + bh * A.track_ld;
  int32_t* pos_out = A.pos_out + bh * A.track_ld;
  const int64_t since = A.recent_from ? A.recent_from[b] : INT64_MAX;
  // what stays in place; the holes among it are filled by the second kernel
#pragma unroll 4
  for (int i = tid; i < new_len; i += EV_THREADS) {
    const float m = mass[i];
    const int32_t p = spos[i];
    mass_out[i] = m;
    pos_out[i] = p;
  }
  if (len <= keep) {
    if (tid == 0) *plan = EvictPlan{0, new_len, {0, 0}};
    return;
  }
  auto key_of = [&](int i) { return spos[i] >= since ? 0xffffffffu : order_key(mass[i]); };
  // the digit at which the count from above reaches `left`
  auto find_digit = [&](int left) {
    const int d = EV_BINS - 1 - 2 * tid;  // this thread's digits: d, d - 1
    const int n0 = (int)hist[d], n1 = (int)hist[d - 1];
    int all;
    const int before = block_scan(n0 + n1, sums, all);
    if (before < left && left <= before + n0) pick[0] = d, pick[1] = left - before, pick[2] = n0;
    if (before + n0 < left && left <= before + n0 + n1) pick[0] = d - 1, pick[1] = left - before - n0, pick[2] = n1;
    hist[d] = hist[d - 1] = 0;
    __syncthreads();
  };
  const bool whole = len <= EV_PIECE;
#pragma unroll 4
  for (int i = tid; i < len; i += EV_THREADS) {
    const uint32_t k = key_of(i);
    if (whole) keys[i] = k;
    atomicAdd(&hist[k >> 21], 1u);
  }
  __syncthreads();
  find_digit(keep);
  uint32_t thr = (uint32_t)pick[0] << 21;  // kept: keys above, and the first `quota` slots of this key
  int quota = pick[1], tied = pick[2];
#pragma unroll
  for (int shift = 10; shift >= 0 && quota < tied; shift -= 10) {  // (a digit kept whole needs no more)
    const int up = shift + 11 - (shift == 0);
    for (int i = tid; i < len; i += EV_THREADS) {
      const uint32_t k = whole ? keys[i] : key_of(i);
      if (k >> up == thr >> up) atomicAdd(&hist[(k >> shift) & ((1u << (up - shift)) - 1)], 1u);
    }
    __syncthreads();
    find_digit(quota);
    thr |= (uint32_t)pick[0] << shift;
    quota = pick[1];
    tied = pick[2];
    __syncthreads();
  }
  const bool all_ties = quota == tied;  // then thr may be the least key of a digit kept whole: all from it up stay
  int ties = 0, listed = 0;             // running counts over the slots so far
  for (int p0 = 0; p0 < len; p0 += EV_PIECE) {
    const int n = min(EV_PIECE, len - p0), c = ((n + EV_THREADS - 1) / EV_THREADS) | 1;
    if (!whole) {
      __syncthreads();
      for (int i = tid; i < n; i += EV_THREADS) keys[i] = key_of(p0 + i);
    }
    __syncthreads();
    const int i0 = min(n, tid * c), i1 = min(n, i0 + c);  // this thread's slots (c odd: no bank is hit twice)
    int rank = 0, total;
    if (!all_ties) {
      int mine = 0;
      for (int i = i0; i < i1; ++i) mine += keys[i] == thr;
      rank = ties + block_scan(mine, sums, total);
      ties += total;
    }
    const int rank0 = rank;
    // holes below `keep`, kept slots above it
    auto moves = [&](int i) {
      const uint32_t k = keys[i];
      const bool stay = k > thr || (k == thr && (all_ties || rank++ < quota));
      return stay == (p0 + i >= keep);
    };
    int mine = 0;
    for (int i = i0; i < i1; ++i) mine += moves(i);
    int at = listed + block_scan(mine, sums, total);
    listed += total;
    rank = rank0;
    for (int i = i0; i < i1; ++i)
      if (moves(i)) list[at++] = p0 + i;
  }
  if (tid == 0) *plan = EvictPlan{listed / 2, new_len, {0, 0}};
}

// A thread moves one 16-byte piece of K and of V for EV_MOVES rows at a time.
constexpr int EV_MOVES = 4;
__global__ void __launch_bounds__(256) kv_evict_move_kernel(const KvEvictArgs A) {
  kv_pdl_enter();
  const int hk = blockIdx.y, hkv = A.pool.hkv;
  const int64_t b = blockIdx.z, bh = b * hkv + hk;
  const EvictPlan plan = static_cast<const EvictPlan*>(A.scratch)[bh];
  const int* holes = reinterpret_cast<const int*>(static_cast<const EvictPlan*>(A.scratch) + A.batch * hkv) +
                     bh * evict_list(A.track_ld);
  const int* movers = holes + plan.moves;
  if (blockIdx.x == 0 && hk == 0 && threadIdx.x == 0) A.lens_out[b] = plan.new_len;
  const int ch = A.pool.hd / 8, rows = 256 / ch;  // 16-byte pieces of a row; rows the CTA takes at once
  const int c = threadIdx.x % ch, r = threadIdx.x / ch;
  const int32_t* table = A.table + b * A.table_ld;
  __half* k = static_cast<__half*>(A.pool.k) + 8 * c;
  __half* v = static_cast<__half*>(A.pool.v) + 8 * c;
  for (int m0 = blockIdx.x * rows * EV_MOVES; m0 < plan.moves; m0 += gridDim.x * rows * EV_MOVES) {
    int dst[EV_MOVES], src[EV_MOVES];
    int64_t to[EV_MOVES], from[EV_MOVES];
#pragma unroll
    for (int q = 0; q < EV_MOVES; ++q) {
      const int m = m0 + q * rows + r;
      dst[q] = m < plan.moves ? holes[m] : -1;
      src[q] = m < plan.moves ? movers[m] : -1;
    }
#pragma unroll
    for (int q = 0; q < EV_MOVES; ++q) {
      from[q] = to[q] = -1;
      if (dst[q] < 0) continue;
      from[q] = kv_row(A.pool, table[src[q] / A.pool.page_size], src[q], hk);
      to[q] = kv_row(A.pool, table[dst[q] / A.pool.page_size], dst[q], hk);
      if (from[q] < 0 || to[q] < 0) {
        kv_error(A.err, KV_ERR_PAGE);
        dst[q] = -1;
      }
    }
    uint4 kr[EV_MOVES], vr[EV_MOVES];
    float mass[EV_MOVES];
    int32_t pos[EV_MOVES];
#pragma unroll
    for (int q = 0; q < EV_MOVES; ++q) {
      if (dst[q] < 0) continue;
      kr[q] = *reinterpret_cast<const uint4*>(k + from[q]);
      vr[q] = *reinterpret_cast<const uint4*>(v + from[q]);
      mass[q] = A.mass[bh * A.track_ld + src[q]];
      pos[q] = A.slot_pos[bh * A.track_ld + src[q]];
    }
#pragma unroll
    for (int q = 0; q < EV_MOVES; ++q) {
      if (dst[q] < 0) continue;
      *reinterpret_cast<uint4*>(k + to[q]) = kr[q];
      *reinterpret_cast<uint4*>(v + to[q]) = vr[q];
      if (c == 0) {
        A.mass_out[bh * A.track_ld + dst[q]] = mass[q];
        A.pos_out[bh * A.track_ld + dst[q]] = pos[q];
      }
    }
  }
}

}  // namespace

cudaError_t kv_append(const KvAppendArgs& a, cudaStream_t s) {
  const bool vec_in = reinterpret_cast<uintptr_t>(a.qkv) % 16 == 0 && a.ld % 4 == 0;
  const bool vec_out = reinterpret_cast<uintptr_t>(a.q_out) % 16 == 0 && a.q_ld % 4 == 0;
  return launch_pdl(kv_append_kernel, dim3((unsigned)a.rows), dim3(AP_THREADS), 0, s, a, vec_in, vec_out);
}

size_t kv_evict_scratch_bytes(int64_t batch, int hkv, int64_t track_ld) {
  return (size_t)batch * hkv * (sizeof(EvictPlan) + (size_t)evict_list(track_ld) * sizeof(int));
}

cudaError_t kv_evict_init_device() {
  return cudaFuncSetAttribute(kv_evict_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)EV_SMEM);
}

cudaError_t kv_evict(const KvEvictArgs& a, int* launches, cudaStream_t s) {
  const int64_t most = std::min(a.track_ld, a.table_ld * a.pool.page_size);  // slots a sequence may have
  const size_t smem = (size_t)std::min<int64_t>(most, EV_PIECE) * 4;
  cudaError_t e = launch_pdl(kv_evict_select_kernel, dim3((unsigned)a.pool.hkv, (unsigned)a.batch), dim3(EV_THREADS),
                             smem, s, a);
  if (e != cudaSuccess) return e;
  const int64_t moves = std::min<int64_t>(a.keep, std::max<int64_t>(0, most - a.keep));
  const int64_t per_cta = 256 / (a.pool.hd / 8) * EV_MOVES;
  const unsigned ctas = (unsigned)std::max<int64_t>(1, std::min<int64_t>((moves + per_cta - 1) / per_cta, 64));
  *launches = 1;
  e = launch_pdl(kv_evict_move_kernel, dim3(ctas, (unsigned)a.pool.hkv, (unsigned)a.batch), dim3(256), 0, s, a);
  *launches += e == cudaSuccess;
  return e;
}

}  // namespace kq
