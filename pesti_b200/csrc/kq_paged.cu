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
// One CTA per row, one thread per (head, pair): q and k turned, k and v rounded
// to f16 into their slot.
__global__ void __launch_bounds__(256) kv_append_kernel(const KvAppendArgs A) {
  kv_pdl_enter();
  const int half = A.pool.hd / 2, hkv = A.pool.hkv;
  const int64_t r = blockIdx.x;
  const int32_t slot = A.slots[r];
  if (slot < 0) return;
  const int64_t b = A.seqs ? A.seqs[r] : r;
  if (b < 0 || b >= A.batch || slot >= A.table_ld * A.pool.page_size || (A.slot_pos && slot >= A.track_ld)) {
    if (threadIdx.x == 0) kv_error(A.err, KV_ERR_ROW);
    return;
  }
  const int32_t pos = A.pos ? A.pos[r] : slot;
  const int32_t page = A.table[b * A.table_ld + slot / A.pool.page_size];
  const bool bad = page < 0 || page >= A.pool.pages;
  if (bad && threadIdx.x == 0) kv_error(A.err, KV_ERR_PAGE);
  const float* row = A.qkv + r * A.ld;
  __half* kc = static_cast<__half*>(A.pool.k);
  __half* vc = static_cast<__half*>(A.pool.v);
  for (int e = threadIdx.x; e < (A.hq + hkv) * half; e += blockDim.x) {
    const int head = e / half, i = e - head * half;
    float c, s;
    rope_turn(pos, i, half, A.log2_theta, c, s);
    const float x = row[(int64_t)head * A.pool.hd + i], y = row[(int64_t)head * A.pool.hd + i + half];
    if (head < A.hq) {
      if (!A.q_out) continue;
      float* o = A.q_out + r * A.q_ld + (int64_t)head * A.pool.hd;
      o[i] = x * c - y * s;
      o[i + half] = x * s + y * c;
    } else if (!bad) {
      const int h = head - A.hq;
      const float* v = row + (int64_t)(A.hq + hkv + h) * A.pool.hd;
      const int64_t o = kv_row(A.pool, page, slot, h);
      kc[o + i] = __float2half_rn(x * c - y * s);
      kc[o + i + half] = __float2half_rn(x * s + y * c);
      vc[o + i] = __float2half_rn(v[i]);
      vc[o + i + half] = __float2half_rn(v[i + half]);
    }
  }
  if (A.slot_pos)
    for (int h = threadIdx.x; h < hkv; h += blockDim.x) A.slot_pos[(b * hkv + h) * A.track_ld + slot] = pos;
}

// ---- eviction ---------------------------------------------------------------------
// Kept are the `keep` slots that come first in the order (protected slots, then
// by mass descending, ties by slot).  Attention does not depend on the order of
// the slots, so only the holes below `keep` are filled, in ascending order, with
// the kept slots above it: the fewest rows move, and no row that is read is
// written.
constexpr int EV_THREADS = 1024, EV_ITEMS = 4;

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
  kv_pdl_enter();
  __shared__ unsigned hist[256];
  __shared__ int sums[32];
  __shared__ uint32_t pick[2];  // digit, how many of it still to keep
  const int hk = blockIdx.x, hkv = A.pool.hkv, tid = threadIdx.x;
  const int64_t b = blockIdx.y, bh = b * hkv + hk;
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
  auto key_of = [&](int i) { return spos[i] >= since ? 0xffffffffu : order_key(mass[i]); };
  // the key of the last slot kept, and how many slots with that key are
  uint32_t thr = 0;
  int quota = len;
  if (len > keep) {
    uint32_t prefix = 0;
    int left = keep;
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int e = tid; e < 256; e += EV_THREADS) hist[e] = 0;
      __syncthreads();
      for (int i = tid; i < len; i += EV_THREADS) {
        const uint32_t k = key_of(i);
        if (shift == 24 || (k >> (shift + 8)) == prefix) atomicAdd(&hist[(k >> shift) & 255u], 1u);
      }
      __syncthreads();
      if (tid == 0) {
        int d = 255;
        while (d > 0 && (int)hist[d] < left) left -= hist[d--];
        pick[0] = d;
        pick[1] = left;
      }
      __syncthreads();
      prefix = prefix << 8 | pick[0];
      left = pick[1];
      __syncthreads();
    }
    thr = prefix;
    quota = left;
  }
  int ties = 0, listed = 0;  // running counts over the slots so far
  for (int c0 = 0; c0 < len; c0 += EV_THREADS * EV_ITEMS) {
    const int i0 = c0 + tid * EV_ITEMS;
    uint32_t key[EV_ITEMS];
    int tie = 0;
#pragma unroll
    for (int j = 0; j < EV_ITEMS; ++j) {
      key[j] = i0 + j < len ? key_of(i0 + j) : 0u;
      tie += i0 + j < len && key[j] == thr;
    }
    int tie_total, total;
    int rank = ties + block_scan(tie, sums, tie_total);
    bool stay[EV_ITEMS];
    int mine = 0;
#pragma unroll
    for (int j = 0; j < EV_ITEMS; ++j) {
      const int i = i0 + j;
      stay[j] = i < len && (key[j] > thr || (key[j] == thr && rank < quota));
      rank += i < len && key[j] == thr;
      mine += i < len && (i < keep ? !stay[j] : stay[j]);
    }
    int at = listed + block_scan(mine, sums, total);
#pragma unroll
    for (int j = 0; j < EV_ITEMS; ++j) {
      const int i = i0 + j;
      if (i >= len) break;
      if (i < keep) {
        if (stay[j]) {
          mass_out[i] = mass[i];
          pos_out[i] = spos[i];
        } else {
          list[at++] = i;
        }
      } else if (stay[j]) {
        list[at++] = i;
      }
    }
    ties += tie_total;
    listed += total;
  }
  if (tid == 0) *plan = EvictPlan{listed / 2, new_len, {0, 0}};
}

__global__ void __launch_bounds__(256) kv_evict_move_kernel(const KvEvictArgs A) {
  kv_pdl_enter();
  const int hk = blockIdx.y, hkv = A.pool.hkv;
  const int64_t b = blockIdx.z, bh = b * hkv + hk;
  const EvictPlan plan = static_cast<const EvictPlan*>(A.scratch)[bh];
  const int* holes = reinterpret_cast<const int*>(static_cast<const EvictPlan*>(A.scratch) + A.batch * hkv) +
                     bh * evict_list(A.track_ld);
  const int* movers = holes + plan.moves;
  if (blockIdx.x == 0 && hk == 0 && threadIdx.x == 0) A.lens_out[b] = plan.new_len;
  const int ch = A.pool.hd / 8;  // 16-byte pieces of a row
  const int32_t* table = A.table + b * A.table_ld;
  for (int e = blockIdx.x * blockDim.x + threadIdx.x; e < plan.moves * ch; e += gridDim.x * blockDim.x) {
    const int m = e / ch, c = e - m * ch, dst = holes[m], src = movers[m];
    const int64_t from = kv_row(A.pool, table[src / A.pool.page_size], src, hk);
    const int64_t to = kv_row(A.pool, table[dst / A.pool.page_size], dst, hk);
    if (from < 0 || to < 0) {
      kv_error(A.err, KV_ERR_PAGE);
      continue;
    }
    __half* k = static_cast<__half*>(A.pool.k);
    __half* v = static_cast<__half*>(A.pool.v);
    reinterpret_cast<uint4*>(k + to)[c] = reinterpret_cast<const uint4*>(k + from)[c];
    reinterpret_cast<uint4*>(v + to)[c] = reinterpret_cast<const uint4*>(v + from)[c];
    if (c == 0) {
      A.mass_out[bh * A.track_ld + dst] = A.mass[bh * A.track_ld + src];
      A.pos_out[bh * A.track_ld + dst] = A.slot_pos[bh * A.track_ld + src];
    }
  }
}

}  // namespace

cudaError_t kv_append(const KvAppendArgs& a, cudaStream_t s) {
  return launch_pdl(kv_append_kernel, dim3((unsigned)a.rows), dim3(256), 0, s, a);
}

size_t kv_evict_scratch_bytes(int64_t batch, int hkv, int64_t track_ld) {
  return (size_t)batch * hkv * (sizeof(EvictPlan) + (size_t)evict_list(track_ld) * sizeof(int));
}

cudaError_t kv_evict(const KvEvictArgs& a, int* launches, cudaStream_t s) {
  dim3 grid((unsigned)a.pool.hkv, (unsigned)a.batch);
  cudaError_t e = launch_pdl(kv_evict_select_kernel, grid, dim3(EV_THREADS), 0, s, a);
  if (e != cudaSuccess) return e;
  *launches = 2;
  return launch_pdl(kv_evict_move_kernel, dim3(16, (unsigned)a.pool.hkv, (unsigned)a.batch), dim3(256), 0, s, a);
}

}  // namespace kq
