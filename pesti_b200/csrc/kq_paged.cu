// kq_paged.cu -- a paged f16 key-value cache: appending rows and eviction by
// accumulated attention weight (include/pesti_decoder.h, kq_kv_append and
// kq_kv_evict).
#include "kq_paged.cuh"

#include <cooperative_groups.h>
#include <cuda_fp16.h>
#include <math.h>

#include <algorithm>

namespace kq {
namespace {

namespace cg = cooperative_groups;

// ---- append ---------------------------------------------------------------------
// 16 to 256 threads per row, by its length: the row's angles once (in 64 bits, hd / 2
// of them, from frequencies that the CTA works out before its rows arrive) into
// shared memory, then four consecutive pairs of a head per thread and step.  Bound
// by the row's bytes: f32 in, f32 q and f16 k, v out.  Many small CTAs hide the chain
// slot - page - row better than several steps' loads in flight: 4099 rows of 32 / 8
// heads of 128 took 33.2 us with one step and eight CTAs per SM, 38.9 with four steps
// and four (34.9 us, 5290 GB/s, since keys are exact and heads found by shifts).
constexpr int AP_THREADS = 256, AP_MAX_HALF = 128;

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
__device__ __forceinline__ uint32_t pair_bits(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint2 halves(float4 v) { return make_uint2(pair_bits(v.x, v.y), pair_bits(v.z, v.w)); }

// Two pairs of a key turned and rounded to f16 as turn_key's are: in plain f32, and
// where its error could round another way (one pair in 100) by exact_dot2.  The error:
// c, s, the product rounded by itself and the sum each add 2^-24 of what they round,
// together at most 3 x 2^-24 of the two products.  lo: what f32 leaves of the cosines,
// and `half` behind that of the sines.  (4099 rows: 1.0 us less of 37.6 than by exact_dot2 alone.)
__device__ __forceinline__ void turn_keys(float2 x, float2 y, float2 c, float2 s, const float* lo, int half,
                                          uint32_t& a, uint32_t& b) {
  constexpr float E = 0x1.8p-23f;
  // x c + y s of both pairs, as two f16
  auto dots = [&](float2 y, float2 c, const float* c_lo, float2 s, const float* s_lo) {
    const float p0 = x.x * c.x, p1 = x.y * c.y;
    const float a0 = fmaf(y.x, s.x, p0), a1 = fmaf(y.y, s.y, p1);
    const float e0 = E * fmaf(fabsf(y.x), fabsf(s.x), fabsf(p0)), e1 = E * fmaf(fabsf(y.y), fabsf(s.y), fabsf(p1));
    const uint32_t least = pair_bits(a0 - e0, a1 - e1);
    if (least == pair_bits(a0 + e0, a1 + e1)) return least;
    return pair_bits(exact_dot2(x.x, c.x, c_lo[0], y.x, s.x, s_lo[0]), exact_dot2(x.y, c.y, c_lo[1], y.y, s.y, s_lo[1]));
  };
  a = dots(make_float2(-y.x, -y.y), c, lo, s, lo + half);
  b = dots(y, s, lo + half, c, lo);
}

template <int TPR>
__global__ void __launch_bounds__(AP_THREADS, 8) kv_append_kernel(const KvAppendArgs A, bool vec_in, bool vec_out) {
  extern __shared__ float4 turns[];  // per row of the CTA: hd / 2 cosines, as many sines, and what f32 leaves of both
  __shared__ double freq[AP_MAX_HALF];
  const int hd = A.pool.hd, half = hd / 2, hkv = A.pool.hkv, tid = threadIdx.x % TPR;
  if (threadIdx.x < half) freq[threadIdx.x] = rope_freq(threadIdx.x, half, A.log2_theta);
  __syncthreads();
  kv_pdl_enter();
  const int64_t r = (int64_t)blockIdx.x * (AP_THREADS / TPR) + threadIdx.x / TPR;
  float4* turn_c = turns + (threadIdx.x / TPR) * half;
  float4* turn_s = turn_c + half / 4;
  // q and k heads in quads of pairs (q only where it is wanted); the first loads come
  // before the row's place is known
  const float* row = A.qkv + r * A.ld;
  const int quads = half / 4, log2_quads = 31 - __clz(quads);  // of a head: 8, 16 or 32
  const int first = A.q_out ? 0 : A.hq * quads, end = r < A.rows ? (A.hq + hkv) * quads : 0;
  float4 x, y;
  auto load = [&](int e) {
    if (e >= end) return;
    const float* p = row + (int64_t)(e >> log2_quads) * hd + 4 * (e & (quads - 1));
    x = load4(p, vec_in);
    y = load4(p + half, vec_in);
  };
  load(first + tid);
  const int32_t slot = r < A.rows ? A.slots[r] : -1;
  const int64_t b = slot >= 0 && A.seqs ? A.seqs[r] : r;
  const bool bad = slot < -1 || (slot >= 0 && (b < 0 || b >= A.batch || slot >= A.table_cols * A.pool.page_size ||
                                               ((A.slot_pos || A.mass) && slot >= A.track_ld)));
  if (bad && tid == 0) kv_error(A.bad, KV_ERR_ROW);
  const bool live = slot >= 0 && !bad;
  int32_t pos = 0;
  int64_t row0 = -1;
  if (live) {
    const int32_t page = A.table[b * A.table_ld + slot / A.pool.page_size];
    pos = A.pos ? A.pos[r] : slot;
    for (int i = tid; i < half; i += TPR) {
      double c, s;
      rope_turn(pos, freq[i], c, s);
      float* to = reinterpret_cast<float*>(turn_c) + i;
      to[0] = (float)c;
      to[half] = (float)s;
      to[2 * half] = (float)(c - (double)to[0]);
      to[3 * half] = (float)(s - (double)to[half]);
    }
    row0 = kv_row(A.pool, page, slot, 0);
    if (row0 < 0 && tid == 0) kv_error(A.bad, KV_ERR_PAGE);
  }
  __syncthreads();
  if (!live) return;
  const int64_t head_ld = (int64_t)A.pool.page_size * hd;
  float* q_out = A.q_out ? A.q_out + r * A.q_ld : nullptr;
  __half* kc = static_cast<__half*>(A.pool.k) + row0;
  __half* vc = static_cast<__half*>(A.pool.v) + row0;
  for (int e = first + tid; e < end; e += TPR) {
    if (e != first + tid) load(e);
    const int head = e >> log2_quads, i = 4 * (e & (quads - 1));
    const float4 c = turn_c[i / 4], s = turn_s[i / 4];
    if (head < A.hq) {
      const float4 a = make_float4(x.x * c.x - y.x * s.x, x.y * c.y - y.y * s.y, x.z * c.z - y.z * s.z,
                                   x.w * c.w - y.w * s.w);
      const float4 d = make_float4(x.x * s.x + y.x * c.x, x.y * s.y + y.y * c.y, x.z * s.z + y.z * c.z,
                                   x.w * s.w + y.w * c.w);
      float* o = q_out + (int64_t)head * hd + i;
      store4(o, a, vec_out);
      store4(o + half, d, vec_out);
    } else if (row0 >= 0) {
      const float* lo = reinterpret_cast<const float*>(turn_c) + 2 * half + i;
      uint2 a, d;
      turn_keys(make_float2(x.x, x.y), make_float2(y.x, y.y), make_float2(c.x, c.y), make_float2(s.x, s.y), lo, half,
                a.x, d.x);
      turn_keys(make_float2(x.z, x.w), make_float2(y.z, y.w), make_float2(c.z, c.w), make_float2(s.z, s.w), lo + 2,
                half, a.y, d.y);
      __half* o = kc + (head - A.hq) * head_ld + i;
      *reinterpret_cast<uint2*>(o) = a;
      *reinterpret_cast<uint2*>(o + half) = d;
    }
  }
  if (row0 < 0) return;
  for (int e = tid; e < hkv * (hd / 4); e += TPR) {
    const int h = e >> (log2_quads + 1), i = 4 * (e & (2 * quads - 1));
    *reinterpret_cast<uint2*>(vc + h * head_ld + i) = halves(load4(row + (int64_t)(A.hq + hkv + h) * hd + i, vec_in));
  }
  for (int h = tid; h < hkv; h += TPR) {
    const int64_t at = (b * hkv + h) * A.track_ld + slot;
    if (A.mass) A.mass[at] = 0.f;
    if (A.slot_pos) A.slot_pos[at] = pos;
  }
}

// ---- eviction ---------------------------------------------------------------------
// Kept are the `keep` slots that come first in the order (protected slots, then
// by mass descending, ties by slot).  Attention does not depend on the order of
// the slots, so only the holes below `keep` are filled, in ascending order, with
// the kept slots above it: the fewest rows move, and no row that is read is
// written.
//
// A cluster of up to eight CTAs selects for a (sequence, kv head), each for its
// share of the slots: the key of the last slot kept by three passes over 11-bit
// digits whose counts every CTA reads from the others' shared memory, then the
// lists of holes and kept slots above by sums over the threads, each owning
// consecutive slots as bits of a mask.  Keys are read from global memory once and
// stay in shared memory (up to EV_PIECE slots a CTA; longer shares go piece by
// piece).  A second kernel moves the rows: it is bound by them, the first by the
// latency of its passes.  Measured: 8 sequences of 2113 to 2048 slots, 8 heads of 128,
// 13.7 us; 4 of up to 32,771 to 4096 31.4 us, of which the rows take about half (33 MB
// read, as much written).
constexpr int EV_THREADS = 512, EV_BINS = 2048, EV_PIECE = 20480, EV_LOADS = 8, EV_MAX_CLUSTER = 8;
constexpr size_t EV_SMEM = (size_t)EV_PIECE * 4;

// f32 -> unsigned with the same order; -0 as 0, NaN as -inf
__device__ __forceinline__ uint32_t order_key(float f) {
  const uint32_t u = __float_as_uint(isnan(f) ? -INFINITY : f + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Exclusive sum over the block; `total` gets the sum.
__device__ __forceinline__ int block_scan(int v, int* warp_sums, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto scan = [&](int x) {  // inclusive, over the warp
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    return x;
  };
  const int x = scan(v);
  __syncthreads();
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  const int w = lane < EV_THREADS / 32 ? warp_sums[lane] : 0, upto = scan(w);
  total = __shfl_sync(0xffffffffu, upto, 31);
  return __shfl_sync(0xffffffffu, upto - w, warp) + x - v;
}

struct EvictPlan {  // one (sequence, kv head)
  int moves, new_len;
  int pad[2];
};

// Per (sequence, kv head) after the plans: the holes, then as many movers (holes
// lie below `keep`, movers above it: together at most track_ld).
__host__ __device__ __forceinline__ int64_t evict_list(int64_t track_ld) { return (track_ld + 3) & ~int64_t(3); }

struct EvictShared {
  alignas(16) unsigned hist[EV_BINS];
  int sums[32];
  int pick[3];                // digit, how many of it are kept, how many there are
  int sum[EV_MAX_CLUSTER];    // counts of every CTA's digits
  int tot[2][EV_MAX_CLUSTER];  // ties and listed slots of every CTA
};

__global__ void __launch_bounds__(EV_THREADS, 2) kv_evict_select_kernel(const KvEvictArgs A) {
  extern __shared__ uint32_t keys[];
  __shared__ EvictShared S;
  cg::cluster_group cluster = cg::this_cluster();
  const int CL = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
  const int hk = blockIdx.x / CL, hkv = A.pool.hkv, tid = threadIdx.x;
  const int64_t b = blockIdx.y, bh = b * hkv + hk;
  for (int e = tid; e < EV_BINS; e += EV_THREADS) S.hist[e] = 0;
  __syncthreads();
  kv_pdl_enter();
  bool bad;
  const int len = (int)kv_len(A.lens[b], min(A.table_cols * A.pool.page_size, A.track_ld), &bad);
  if (bad && tid == 0) kv_error(A.bad, KV_ERR_LEN);
  const int keep = A.keep, new_len = min(len, keep);
  const int share = (int)(((int64_t)len + CL - 1) / CL), s0 = min(len, part * share), n = min(len, s0 + share) - s0;
  EvictPlan* plan = static_cast<EvictPlan*>(A.scratch) + bh;
  int* list = reinterpret_cast<int*>(static_cast<EvictPlan*>(A.scratch) + A.batch * hkv) + bh * evict_list(A.track_ld);
  const float* mass = A.mass + bh * A.track_ld + s0;
  const int32_t* spos = A.slot_pos + bh * A.track_ld + s0;
  float* mass_out = A.mass_out + bh * A.track_ld + s0;
  int32_t* pos_out = A.pos_out + bh * A.track_ld + s0;
  const int64_t since = A.recent_from ? A.recent_from[b] : INT64_MAX;
  // what stays in place; the holes among it are filled by the second kernel
  auto stays_put = [&](int i, float m, int32_t p) {
    if (s0 + i >= new_len) return;
    mass_out[i] = m;
    pos_out[i] = p;
  };
  auto key_of = [&](float m, int32_t p) { return p >= since ? 0xffffffffu : order_key(m); };
  // f(slot, mass, position) over this CTA's slots, EV_LOADS of each in flight per thread
  auto each = [&](auto f) {
    for (int i = tid; i < n; i += EV_LOADS * EV_THREADS) {
      float m[EV_LOADS];
      int32_t p[EV_LOADS];
#pragma unroll
      for (int q = 0; q < EV_LOADS; ++q)
        if (i + q * EV_THREADS < n) m[q] = mass[i + q * EV_THREADS], p[q] = spos[i + q * EV_THREADS];
#pragma unroll
      for (int q = 0; q < EV_LOADS; ++q)
        if (i + q * EV_THREADS < n) f(i + q * EV_THREADS, m[q], p[q]);
    }
  };
  if (len <= keep) {
    each(stays_put);
    if (part == 0 && tid == 0) *plan = EvictPlan{0, bad ? A.lens[b] : new_len, {0, 0}};
    return;
  }
  auto sync_all = [&] {
    if (CL > 1) cluster.sync();
    else __syncthreads();
  };
  // the digit at which all CTAs' count from above reaches `left`: every CTA joins
  // the counts of its part of the digits (the first has the greatest), the one in
  // whose part it lies finds it
  auto find_digit = [&](int left) {
    sync_all();
    const int digits = EV_BINS / CL, top = EV_BINS - 1 - part * digits;  // this CTA's: [top - digits + 1, top]
    constexpr int MOST = EV_BINS / EV_THREADS;
    const int per = (digits + EV_THREADS - 1) / EV_THREADS;
    int count[MOST] = {}, sum = 0, all;
    if (CL == 1) {
      static_assert(MOST == 4, "16 bytes");
      const uint4 c = reinterpret_cast<const uint4*>(S.hist)[EV_THREADS - 1 - tid];
      count[0] = (int)c.w, count[1] = (int)c.z, count[2] = (int)c.y, count[3] = (int)c.x;
    } else {
#pragma unroll
      for (int q = 0; q < MOST; ++q) {
        const int d = top - tid * per - q;
        if (q >= per || d <= top - digits) continue;
        unsigned c[EV_MAX_CLUSTER];
#pragma unroll
        for (int r = 0; r < EV_MAX_CLUSTER; ++r) c[r] = r < CL ? cluster.map_shared_rank(S.hist, r)[d] : 0;
#pragma unroll
        for (int r = 0; r < EV_MAX_CLUSTER; ++r) count[q] += (int)c[r];
      }
    }
#pragma unroll
    for (int q = 0; q < MOST; ++q) sum += count[q];
    int before = block_scan(sum, S.sums, all), owner = 0;
    if (CL > 1) {
      if (tid < CL) cluster.map_shared_rank(&S, tid)->sum[part] = all;
      cluster.sync();
      int upto = S.sum[0];
      while (upto < left) upto += S.sum[++owner];
      for (int r = 0; r < part; ++r) before += S.sum[r];
    }
#pragma unroll
    for (int q = 0; q < MOST; ++q) {
      if (before < left && left <= before + count[q])
        S.pick[0] = top - tid * per - q, S.pick[1] = left - before, S.pick[2] = count[q];
      before += count[q];
    }
    for (int e = tid; e < EV_BINS; e += EV_THREADS) S.hist[e] = 0;  // (all have read it)
    sync_all();
    const int* pick = CL > 1 ? cluster.map_shared_rank(S.pick, owner) : S.pick;
    return make_int3(pick[0], pick[1], pick[2]);
  };
  const bool whole = n <= EV_PIECE;
  each([&](int i, float m, int32_t p) {
    const uint32_t k = key_of(m, p);
    if (whole) keys[i] = k;
    atomicAdd(&S.hist[k >> 21], 1u);
    stays_put(i, m, p);
  });
  int3 pick = find_digit(keep);
  uint32_t thr = (uint32_t)pick.x << 21;  // kept: keys above, and the first `quota` slots of this key
  int quota = pick.y, tied = pick.z;
#pragma unroll
  for (int shift = 10; shift >= 0 && quota < tied; shift -= 10) {  // (a digit kept whole needs no more)
    const int up = shift + 11 - (shift == 0);
    auto count = [&](uint32_t k) {
      if (k >> up == thr >> up) atomicAdd(&S.hist[(k >> shift) & ((1u << (up - shift)) - 1)], 1u);
    };
    if (whole) {
#pragma unroll 4
      for (int i = tid; i < n; i += EV_THREADS) count(keys[i]);
    } else {
      each([&](int, float m, int32_t p) { count(key_of(m, p)); });
    }
    pick = find_digit(quota);
    thr |= (uint32_t)pick.x << shift;
    quota = pick.y;
    tied = pick.z;
  }
  // This thread's slots of a piece (c <= 41 of them, odd: no bank is hit twice), and
  // the masks of their keys above and at the threshold
  struct Masks {
    int first, n;
    uint64_t above, at_thr;
  };
  auto masks_of = [&](int p0, int rest) {
    const int c = ((rest + EV_THREADS - 1) / EV_THREADS) | 1;
    const int i0 = min(rest, tid * c), m = min(rest, i0 + c) - i0;
    Masks x{p0 + i0, m, 0, 0};
#pragma unroll 4
    for (int j = 0; j < m; ++j) {
      const uint32_t k = keys[i0 + j];
      x.above |= (uint64_t)(k > thr) << j;
      x.at_thr |= (uint64_t)(k == thr) << j;
    }
    return x;
  };
  Masks only{};
  if (whole) only = masks_of(0, n);
  // f(masks) piece by piece
  auto pieces = [&](auto f) {
    if (whole) {
      f(only);
      return;
    }
    for (int p0 = 0; p0 < n; p0 += EV_PIECE) {
      const int rest = min(EV_PIECE, n - p0);
      __syncthreads();
      for (int i = tid; i < rest; i += EV_THREADS) keys[i] = key_of(mass[p0 + i], spos[p0 + i]);
      __syncthreads();
      f(masks_of(p0, rest));
    }
  };
  // What the CTAs before this one count: where its first tie and its first listed
  // slot stand among all.
  auto before_here = [&](int k, int mine) {
    if (CL == 1) return 0;
    if (tid < CL) cluster.map_shared_rank(&S, tid)->tot[k][part] = mine;
    cluster.sync();
    int sum = 0;
    for (int r = 0; r < part; ++r) sum += S.tot[k][r];
    return sum;
  };
  const bool all_ties = quota == tied;  // then thr may be the least key of a digit kept whole: all from it up stay
  int ties = 0, total;
  if (!all_ties) {
    int here = 0;
    pieces([&](Masks x) {
      block_scan(__popcll(x.at_thr), S.sums, total);
      here += total;
    });
    ties = before_here(0, here);
  }
  // the slots that move: holes below `keep`, kept slots above it
  auto movers = [&](auto f) {
    int seen = ties;
    pieces([&](Masks x) {
      if (!all_ties) {  // only the first `quota` of the ties
        const int left = quota - seen - block_scan(__popcll(x.at_thr), S.sums, total);
        seen += total;
        for (int drop = __popcll(x.at_thr) - max(left, 0); drop > 0; --drop)
          x.at_thr &= ~(1ull << (63 - __clzll((long long)x.at_thr)));
      }
      const uint64_t below = (1ull << max(0, min(x.n, keep - s0 - x.first))) - 1;  // slots below `keep`
      f(s0 + x.first, ((1ull << x.n) - 1) & ((x.above | x.at_thr) ^ below));
    });
  };
  int listed = 0;
  auto write = [&](int i0, uint64_t moves, int at) {
    for (; moves; moves &= moves - 1) list[at++] = i0 + __ffsll((long long)moves) - 1;
  };
  if (whole) {
    movers([&](int i0, uint64_t moves) {
      const int at = block_scan(__popcll(moves), S.sums, total);
      listed = before_here(1, total);
      write(i0, moves, listed + at);
      listed += total;
    });
  } else {
    int here = 0;
    movers([&](int, uint64_t moves) {
      block_scan(__popcll(moves), S.sums, total);
      here += total;
    });
    listed = before_here(1, here);
    movers([&](int i0, uint64_t moves) {
      write(i0, moves, listed + block_scan(__popcll(moves), S.sums, total));
      listed += total;
    });
  }
  if (part == CL - 1 && tid == 0) *plan = EvictPlan{listed / 2, new_len, {0, 0}};
}

// A warp moves EV_ROWS rows at a time: half its lanes find where they come from,
// half where they go, then every lane carries 16-byte pieces of K and V.
constexpr int EV_ROWS = 16, EV_MOVERS = 256;
__global__ void __launch_bounds__(EV_MOVERS, 4) kv_evict_move_kernel(const KvEvictArgs A) {
  kv_pdl_enter();
  const int hk = blockIdx.y, hkv = A.pool.hkv, lane = threadIdx.x & 31;
  const int64_t b = blockIdx.z, bh = b * hkv + hk;
  const EvictPlan plan = static_cast<const EvictPlan*>(A.scratch)[bh];
  const int* holes = reinterpret_cast<const int*>(static_cast<const EvictPlan*>(A.scratch) + A.batch * hkv) +
                     bh * evict_list(A.track_ld);
  if (blockIdx.x == 0 && hk == 0 && threadIdx.x == 0) A.lens_out[b] = plan.new_len;
  const int pieces = A.pool.hd / 8, log2_row = 32 - __clz(pieces);  // of K (a power of two); as many of V
  const int32_t* table = A.table + b * A.table_ld;
  const int warps = gridDim.x * (EV_MOVERS / 32);
  for (int m0 = (blockIdx.x * (EV_MOVERS / 32) + (threadIdx.x >> 5)) * EV_ROWS; m0 < plan.moves; m0 += warps * EV_ROWS) {
    const int rows = min(EV_ROWS, plan.moves - m0), mine = lane & (EV_ROWS - 1);
    const bool from = lane >= EV_ROWS;
    const int slot = mine < rows ? holes[(from ? plan.moves : 0) + m0 + mine] : 0;
    const int hole = __shfl_xor_sync(0xffffffffu, slot, EV_ROWS);
    int64_t at = -1;
    if (mine < rows) {
      at = kv_row(A.pool, table[slot / A.pool.page_size], slot, hk);
      if (at < 0) kv_error(A.bad, KV_ERR_PAGE);
      if (from) {  // the mover's weight and position go with its row
        A.mass_out[bh * A.track_ld + hole] = A.mass[bh * A.track_ld + slot];
        A.pos_out[bh * A.track_ld + hole] = A.slot_pos[bh * A.track_ld + slot];
      }
    }
    const int all = rows * 2 * pieces;
    constexpr int AHEAD = 8;
    for (int e0 = 0; e0 < all; e0 += 32 * AHEAD) {
      uint4 v[AHEAD];
      __half* to[AHEAD];
#pragma unroll
      for (int q = 0; q < AHEAD; ++q) {
        const int e = e0 + 32 * q + lane, row = min(e >> log2_row, EV_ROWS - 1), piece = e & (2 * pieces - 1);
        const int64_t src = __shfl_sync(0xffffffffu, at, EV_ROWS + row), dst = __shfl_sync(0xffffffffu, at, row);
        __half* pool = static_cast<__half*>(piece < pieces ? A.pool.k : A.pool.v);
        const int off = 8 * (piece < pieces ? piece : piece - pieces);
        to[q] = e < all && src >= 0 && dst >= 0 ? pool + dst + off : nullptr;
        if (to[q]) v[q] = *reinterpret_cast<const uint4*>(pool + src + off);
      }
#pragma unroll
      for (int q = 0; q < AHEAD; ++q)
        if (to[q]) *reinterpret_cast<uint4*>(to[q]) = v[q];
    }
  }
}

}  // namespace

cudaError_t kv_append(const KvAppendArgs& a, cudaStream_t s) {
  const bool vec_in = reinterpret_cast<uintptr_t>(a.qkv) % 16 == 0 && a.ld % 4 == 0;
  const bool vec_out = reinterpret_cast<uintptr_t>(a.q_out) % 16 == 0 && a.q_ld % 4 == 0;
  // two to four steps a thread
  const int hd = a.pool.hd;
  const int64_t steps = ((a.q_out ? a.hq : 0) + a.pool.hkv) * (hd / 8) + a.pool.hkv * (hd / 4);
  auto launch = [&](auto kernel, int tpr) {
    const int rows = AP_THREADS / tpr;
    return launch_pdl(kernel, dim3((unsigned)((a.rows + rows - 1) / rows)), dim3(AP_THREADS),
                      (size_t)rows * 2 * hd * sizeof(float), s, a, vec_in, vec_out);
  };
  if (steps <= 16 * 4) return launch(kv_append_kernel<16>, 16);
  if (steps <= 32 * 4) return launch(kv_append_kernel<32>, 32);
  if (steps <= 64 * 4) return launch(kv_append_kernel<64>, 64);
  if (steps <= 128 * 4) return launch(kv_append_kernel<128>, 128);
  return launch(kv_append_kernel<256>, 256);
}

size_t kv_evict_scratch_bytes(int64_t batch, int hkv, int64_t track_ld) {
  if (kv_too_many(batch * hkv, track_ld, (int64_t)(sizeof(EvictPlan) + 4 * sizeof(int)))) return SIZE_MAX;
  return (size_t)batch * hkv * (sizeof(EvictPlan) + (size_t)evict_list(track_ld) * sizeof(int));
}

cudaError_t kv_evict_init_device() {
  return cudaFuncSetAttribute(kv_evict_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)EV_SMEM);
}

cudaError_t kv_evict(const KvEvictArgs& a, int* launches, cudaStream_t s) {
  const int64_t most = std::min(a.track_ld, a.table_cols * a.pool.page_size);  // slots a sequence may have
  const int64_t pairs = a.batch * a.pool.hkv;
  // more CTAs per pair while each has over eight slots a thread and SMs are left (two
  // barriers of the cluster per digit cost what a CTA alone needs for about as many)
  int cl = 1;
  while (cl < EV_MAX_CLUSTER && most > cl * 8 * EV_THREADS && pairs * cl <= a.num_sms) cl *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.pool.hkv * cl), (unsigned)a.batch);
  cfg.blockDim = dim3(EV_THREADS);
  cfg.dynamicSmemBytes = (size_t)std::min<int64_t>((most + cl - 1) / cl, EV_PIECE) * 4;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cl;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kv_evict_select_kernel, a);
  if (e != cudaSuccess) return e;
  // a warp per EV_ROWS rows, up to about eight CTAs per SM over all pairs
  const int64_t moves = std::min<int64_t>(a.keep, std::max<int64_t>(0, most - a.keep));
  const int64_t per_cta = EV_MOVERS / 32 * EV_ROWS, cap = std::max<int64_t>(1, 8 * a.num_sms / pairs);
  const unsigned ctas = (unsigned)std::max<int64_t>(1, std::min<int64_t>((moves + per_cta - 1) / per_cta, cap));
  *launches = 1;
  e = launch_pdl(kv_evict_move_kernel, dim3(ctas, (unsigned)a.pool.hkv, (unsigned)a.batch), dim3(EV_MOVERS), 0, s, a);
  *launches += e == cudaSuccess;
  return e;
}

}  // namespace kq
