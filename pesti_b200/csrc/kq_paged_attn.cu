// kq_paged_attn.cu -- attention of one new token per sequence over the paged
// f16 cache (include/pesti_decoder.h, kq_kv_attention and kq_kv_rope_attention).
//
// Mathematics: s_j = q . k_j / sqrt(hd), out = sum_j e^(s_j - M) v_j / sum_j
// e^(s_j - M) in one pass over K and V with a running maximum and sum, in base
// 2 (log2 e is folded into q).  Every K and V byte is used once per query head
// of its group: HBM bounds it.
//
// Split: the (sequence, kv head) pairs' tiles of 64 slots are laid end to end
// and dealt to the CTAs in equal contiguous runs, so ragged batches and one
// long sequence fill the GPU alike.  A CTA walks its run pair by pair; a pair
// that spans CTAs is joined by the last of them to arrive, in slot order (the
// result does not depend on the order of arrival).
//
// Feed: a producer warp brings tiles through a ring in shared memory, one TMA
// box per page piece (a power of two of slots that divides the page, up to 64)
// with the 128-byte swizzle, ids read one tile ahead.
//
// Products: a compute warp owns 16 slots of each tile and keeps its own maximum,
// sum and output until the pair ends, so no barrier among the warps runs per
// tile.  The slots are the M rows of both mma.sync.m16n8k16 products (S^T = K
// q^T and O^T = V^T P^T, f16 in, f32 accumulate) and eight query heads the N
// columns: S^T's accumulators turn into P^T's operand by movmatrix, in
// registers.  q (scaled by a power of two per head) and P enter as two f16
// parts, so that both products keep about 22 bits of their f32 operands; P is
// carried times 2^14, which keeps its second part clear of the subnormals.
// Groups of 9 to 16 heads run a second set of four warps on the same tiles.
//
// Measured: 32 sequences of 128 to 4096 slots, 32 / 8 heads of 128, 53.6 us (264 MB:
// 5.0 TB/s over the call, 7.4 in its steady part; 4.5 us go to lengths - table - first
// tile, about 5 to the join); one of 131,077 slots 91.4 us (5.9 TB/s); one of 2049
// rotated, appended and attended 11.7 us; one of 17, 14 / 2 heads of 64, 4.2 us.
#include "kq_paged.cuh"
#include "kq_sm100.cuh"

#include <cuda_fp16.h>
#include <float.h>
#include <math.h>

namespace kq {
namespace {

using sm100::mbar_arrive;
using sm100::mbar_expect_tx;
using sm100::mbar_wait;
using sm100::smem_u32;

constexpr int PA_TILE = 64;     // slots per ring stage
constexpr int PA_SHIFT = 14;    // P carries 2^14
constexpr int PA_SET = 128;     // threads of the four warps that share a set of eight query heads

template <int HD, int NS>
struct PaCfg {
  static constexpr int KS = HD / 16;  // k16 steps of a row
  static constexpr int CW = 4 * NS, THREADS = (CW + 1) * 32;
  static constexpr int TILE_B = PA_TILE * HD * 2, STAGE = 2 * TILE_B;
  // Two CTAs per SM where two fit with their rings (measured against more, smaller ones: four for
  // 64-dim heads take 30.2 us where two take 24.4, 64 sequences of 2049 with 14 / 2 heads)
  static constexpr int CTAS = HD == 64 || (HD == 128 && NS == 1) ? 2 : 1;
  static constexpr int STAGES = HD == 64 ? 6 : HD == 128 ? (NS == 1 ? 3 : 6) : (NS == 1 ? 3 : 2);
  static constexpr int QF = STAGES * STAGE;            // q fragments [NS][KS][32] {hi, hi, lo, lo}
  static constexpr int RED = QF + NS * KS * 512;       // [NS][2][8][HD] f32: the warps' sums
  static constexpr int ML = RED + NS * 2 * 8 * HD * 4;  // [NS][4][8] {max, sum}
  static constexpr int XS = ML + NS * 4 * 8 * 8;       // [NS][8] 2^e of each head's q
  static constexpr int NEW = XS + NS * 8 * 4;          // [NS][2][HD] f16: the appended row
  static constexpr int BAR = NEW + NS * 2 * HD * 2;    // full, empty
  static constexpr int LAST = BAR + 2 * STAGES * 8;    // [NS][2] flags
  static constexpr int END = LAST + NS * 8;
  static constexpr int PARTS = CTAS * 160;  // CTAs at most, and so parts of a pair
  static_assert(NS * PARTS * 8 * 8 <= QF, "the join's {max, sum} lie in the ring");
  static_assert(END <= 232448 && CTAS * (END + 1024) <= 233472, "shared memory");
};

// Scratch: arrival counters [2 x SMs][2] (zero between calls; one per CTA and
// set: at most one pair begins in a CTA and goes on in the next), the partials'
// {max, sum} and sums [2 x SMs][2][NS][8]([HD]), then for `mass` the final
// {max, sum} [batch][hq] and the scores [batch][hkv][track_ld][GP].  What must
// stay zero does not move with the sizes of a call.
struct PaScratch {
  size_t ml, acc, stats, scores, end;
  __host__ __device__ PaScratch(int64_t batch, int hq, int hkv, int hd, int64_t track, int num_sms) {
    const int64_t slots = 4 * (int64_t)num_sms;
    const int64_t group = hq / hkv, gp = (group + 1) & ~int64_t(1), cols = group > 8 ? 16 : 8;
    ml = ((size_t)slots * sizeof(unsigned) + 255) & ~size_t(255);
    acc = ml + (size_t)slots * cols * 8;
    stats = acc + (size_t)slots * cols * hd * 4;
    scores = stats + (track ? (((size_t)batch * hq * 8 + 255) & ~size_t(255)) : 0);
    end = scores + (size_t)batch * hkv * track * gp * 4;
  }
};

struct PaParams {
  KvAttnArgs a;
  PaScratch at;
  int G, gp, box;    // heads per kv head, that rounded up to even, slots per TMA box
  float scale;
};

__device__ __forceinline__ void bar_set(int set) { asm volatile("bar.sync %0, 128;" ::"r"(1 + set) : "memory"); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void pa_split(float a, float b, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(a, b);
  const __half2 l = __floats2half2_rn(a - __low2float(h), b - __high2float(h));
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}
__device__ __forceinline__ void pa_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void pa_mma0(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {  // C = 0
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void pa_ldm(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void pa_ldm_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t pa_turn(uint32_t x) {  // an 8 x 8 f16 matrix, transposed
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void tma_load_5d(void* dst, const CUtensorMap* map, int row, int head, int page,
                                            uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %2, %4, %5}], "
      "[%6];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(0), "r"(row), "r"(head), "r"(page), "r"(smem_u32(bar))
      : "memory");
}

// Slots a sequence uses: none where its block table (or the tracked slots) cannot hold them.
__device__ __forceinline__ int pa_len(const KvAttnArgs& A, int64_t b, bool* bad) {
  int64_t most = A.table_cols * A.pool.page_size;
  if (A.mass || A.slot_pos) most = min(most, A.track_ld);
  return (int)kv_len(A.lens[b], most, bad);
}
__device__ __forceinline__ int pa_tiles(int len) { return (int)(((int64_t)len + PA_TILE - 1) / PA_TILE); }

// Where a CTA's run stands.  Each pair counts PA_PAIR units before its nt tiles
// (taking up a pair costs a CTA about as much as that many tiles), so that CTAs
// with many short pairs get fewer tiles.
constexpr int PA_PAIR = 2;
struct PaWalk {
  int64_t total, f, f1;  // all units; this CTA's [f, f1)
  int ctas;              // CTAs with units
  int64_t b;
  int hk, len, nt, v;    // the pair, its slots and tiles, and the unit of it that the run stands at

  // Whole warps; every warp of the CTA finds the same place.
  __device__ __forceinline__ void start(const KvAttnArgs& A) {
    const int lane = threadIdx.x & 31, hkv = A.pool.hkv;
    auto units = [&](int64_t i) {
      bool bad;
      const int n = i < A.batch ? pa_tiles(pa_len(A, i, &bad)) : 0;
      return n ? n + PA_PAIR : 0;
    };
    const int first = units(lane);
    int64_t sum = first;
    int pairs = first > 0;
    for (int64_t i = lane + 32; i < A.batch; i += 32) {
      const int n = units(i);
      sum += n;
      pairs += n > 0;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    pairs = __reduce_add_sync(0xffffffffu, pairs);
    total = sum * hkv;
    ctas = (int)min((int64_t)gridDim.x, total);
    // More CTAs shorten the runs and lengthen the joins (a part read costs about an eighth of a tile):
    // the sum is least at sqrt(8 tiles / pair) parts a pair.  Measured for one context of 65,536 and
    // one pair: 45.7, 34.4, 32.7, 34.2, 49.8 us at 1, 4, 8, 16 and no limit; many pairs never reach it.
    ctas = min(ctas, (int)ceilf(sqrtf(8.f * (float)total * (float)((int64_t)pairs * hkv))));
    f = f1 = 0;
    if ((int)blockIdx.x >= ctas) return;
    f = begin(blockIdx.x);
    f1 = begin(blockIdx.x + 1);
    int64_t base = 0;
    for (int64_t b0 = 0;; b0 += 32) {
      const int n = b0 == 0 ? first : units(b0 + lane);
      int64_t incl = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
      }
      const int64_t here = __shfl_sync(0xffffffffu, incl, 31) * hkv;
      if (f < base + here) {
        const int at = __ffs(__ballot_sync(0xffffffffu, f < base + incl * hkv)) - 1;
        const int64_t rem = f - base - __shfl_sync(0xffffffffu, incl - n, at) * hkv;
        const int u = __shfl_sync(0xffffffffu, n, at);
        b = b0 + at;
        hk = (int)div(rem, u);
        v = (int)(rem - (int64_t)hk * u);
        nt = u - PA_PAIR;
        bool bad;
        len = pa_len(A, b, &bad);
        return;
      }
      base += here;
    }
  }
  // a / b; 64-bit division is a long sequence of instructions, rarely needed
  static __device__ __forceinline__ int64_t div(int64_t a, int64_t b) {
    return (uint64_t)(a | b) >> 32 ? a / b : (int64_t)((uint32_t)a / (uint32_t)b);
  }
  __device__ __forceinline__ int64_t begin(int cta) const { return div(total * cta, ctas); }
  __device__ __forceinline__ int owner(int64_t unit) const { return (int)div((unit + 1) * ctas - 1, total); }
  __device__ __forceinline__ int here() const { return (int)min((int64_t)(nt + PA_PAIR - v), f1 - f); }
  __device__ __forceinline__ int j0() const { return max(0, v - PA_PAIR); }        // this CTA's tiles of the pair:
  __device__ __forceinline__ int j1() const { return max(0, v + here() - PA_PAIR); }  // [j0, j1), j1 <= nt
  // first and last CTA with tiles of the pair
  __device__ __forceinline__ int c0() const { return owner(f - v + PA_PAIR); }
  __device__ __forceinline__ int c1() const { return owner(f - v + PA_PAIR + nt - 1); }
  // on to the run's next pair; false (and f = f1) at its end
  __device__ __forceinline__ bool next(const KvAttnArgs& A) {
    f += here();
    if (f >= f1) return false;
    v = 0;
    if (++hk < A.pool.hkv) return true;
    hk = 0;
    bool bad;
    do {
      ++b;  // f < total: a sequence with slots follows
      len = pa_len(A, b, &bad);
    } while (len == 0);
    nt = pa_tiles(len);
    return true;
  }
  // past pairs of which this CTA has no tile
  __device__ __forceinline__ bool settle(const KvAttnArgs& A) {
    bool more = f < f1;
    while (more && j0() >= j1()) more = next(A);
    return more;
  }
};

template <int HD, int NS>
__global__ void __launch_bounds__(PaCfg<HD, NS>::THREADS, PaCfg<HD, NS>::CTAS)
    kv_attn_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                   const __grid_constant__ PaParams P) {
  using C = PaCfg<HD, NS>;
  constexpr int HALF = HD / 2;
  extern __shared__ __align__(1024) uint8_t sm[];
  const KvAttnArgs& A = P.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint64_t* full = reinterpret_cast<uint64_t*>(sm + C::BAR);
  uint64_t* empty = full + C::STAGES;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (tid == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      sm100::mbar_init(full + s, 1);
      sm100::mbar_init(empty + s, C::CW);
    }
    sm100::mbar_fence_init();
  }
  __syncthreads();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  PaWalk W;
  W.start(A);
  bool more = W.settle(A);

  if (warp == C::CW) {
    // ---- producer ----
    const bool is_v = lane >= 16;
    const int i = lane & 15, boxes = PA_TILE / P.box;
    int it = 0;
    bool live = true;
    while (more && live) {
      const int32_t* table = A.table + W.b * A.table_ld;
      const int j1 = W.j1();
      auto id_of = [&](int j, int& page, int& row) {
        const int64_t slot = (int64_t)j * PA_TILE + (int64_t)i * P.box;
        page = row = 0;
        if (i < boxes && slot < W.len) {
          page = table[slot / A.pool.page_size];
          row = (int)(slot % A.pool.page_size);
        }
      };
      int page, row;
      id_of(W.j0(), page, row);
      for (int j = W.j0(); j < j1; ++j, ++it) {
        const int64_t slot0 = (int64_t)j * PA_TILE;
        const int valid = (int)min((int64_t)boxes, (W.len - slot0 + P.box - 1) / P.box);
        const int s = it % C::STAGES;
        const int page_now = page, row_now = row;
        if (j + 1 < j1) id_of(j + 1, page, row);
        if (it >= C::STAGES)
          live = __all_sync(0xffffffffu, mbar_wait(empty + s, (it / C::STAGES - 1) & 1, A.err, KV_ERR_WAIT));
        if (!live) break;
        if (lane == 0) mbar_expect_tx(full + s, (uint32_t)valid * 2 * P.box * HD * 2);
        __syncwarp();
        if (i < valid) {
          // a page outside the pool is outside the descriptor: the box is filled with zeros
          if (page_now < 0 || page_now >= A.pool.pages) kv_error(A.bad, KV_ERR_PAGE);
          tma_load_5d(sm + s * C::STAGE + (is_v ? C::TILE_B : 0) + i * P.box * HD * 2, is_v ? &vmap : &kmap, row_now,
                      W.hk, page_now, full + s);
        }
      }
      more = W.next(A) && W.settle(A);
    }
    // no copy may be in flight when the CTA retires
    for (int k = max(0, it - C::STAGES); k < it; ++k) mbar_wait(full + k % C::STAGES, (k / C::STAGES) & 1, A.err, KV_ERR_WAIT);
    return;
  }

  // ---- compute ----
  const int set = warp >> 2, w = warp & 3, stid = tid - set * PA_SET;
  const int g = lane >> 2, c = lane & 3;
  const int hkv = A.pool.hkv, h0 = 8 * set, nh = min(8, P.G - h0);  // this set's query heads of a group
  float* red = reinterpret_cast<float*>(sm + C::RED) + set * 2 * 8 * HD;
  uint32_t* qf = reinterpret_cast<uint32_t*>(sm + C::QF) + set * C::KS * 128;
  float2* ml_s = reinterpret_cast<float2*>(sm + C::ML) + set * 32;
  float* xs_s = reinterpret_cast<float*>(sm + C::XS) + set * 8;
  __half* new_s = reinterpret_cast<__half*>(sm + C::NEW) + set * 2 * HD;
  int* last_s = reinterpret_cast<int*>(sm + C::LAST) + 2 * set;
  char* scratch = static_cast<char*>(A.scratch);
  unsigned* ctr = reinterpret_cast<unsigned*>(scratch);
  float2* part_ml = reinterpret_cast<float2*>(scratch + P.at.ml);
  float* part = reinterpret_cast<float*>(scratch + P.at.acc);
  float2* stats = reinterpret_cast<float2*>(scratch + P.at.stats);
  float* scores = reinterpret_cast<float*>(scratch + P.at.scores);

  // idle rows: zeros
  for (int64_t b = blockIdx.x; b < A.batch; b += gridDim.x) {
    bool bad;
    if (pa_len(A, b, &bad) == 0)
      for (int e = tid; e < A.hq * HD; e += C::CW * 32) A.out[b * A.out_ld + e] = 0.f;
    if (bad && tid == 0) kv_error(A.bad, KV_ERR_LEN);
  }

  // lane's places in a 16-slot group, swizzled: rows of K (M rows, two k8 halves) and of V
  // (transposed); the 16-byte piece 2 kk of a 128-byte row is then one xor away
  const uint32_t k_row = (lane & 7) + ((lane >> 3) & 1) * 8, v_row = (lane & 7) + (lane >> 4) * 8;
  const uint32_t k_lane = k_row * 128 + (((lane >> 4) ^ (lane & 7)) << 4);
  const uint32_t v_lane = v_row * 128 + ((((lane >> 3) & 1) ^ (lane & 7)) << 4);
  const uint32_t box_b = P.box * 128;  // bytes of one 64-dim half of a box
  const uint32_t group_off = (uint32_t)(16 * w / P.box) * P.box * HD * 2 + (uint32_t)(16 * w % P.box) * 128;
  const uint32_t ring = smem_u32(sm) + group_off;

  // q of the set's heads 2w, 2w + 1: a lane holds dims i, i + 1 and their partners
  // i + HD/2, i + HD/2 + 1 of IN pieces per head (HD 64: half a warp per head)
  constexpr int IN = HD == 256 ? 2 : 1, HEADS = HD == 64 ? 1 : 2;
  const int qi = HD == 64 ? 2 * (lane & 15) : 2 * lane;
  const int qh = HD == 64 ? 2 * w + (lane >> 4) : 2 * w;
  float qr[HEADS][IN][4], nr[IN][4];
  int32_t pos = 0, new_page = -1;
  auto load_q = [&](const PaWalk& at) {
    if (A.rope) pos = A.pos ? A.pos[at.b] : at.len - 1;
    const float* row = A.q + at.b * A.q_ld;
#pragma unroll
    for (int h = 0; h < HEADS; ++h)
#pragma unroll
      for (int k = 0; k < IN; ++k) {
        const float* p = row + (int64_t)(at.hk * P.G + h0 + qh + h) * HD + qi + 64 * k;
#pragma unroll
        for (int e = 0; e < 4; ++e) qr[h][k][e] = qh + h < nh ? p[(e & 1) + (e >> 1) * HALF] : 0.f;
      }
    if (A.rope && w < 2 && at.j1() == at.nt) {  // the new k (warp 0) and v (warp 1)
      const float* p = row + (int64_t)(A.hq + w * hkv + at.hk) * HD + qi;
#pragma unroll
      for (int k = 0; k < IN; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) nr[k][e] = p[64 * k + (e & 1) + (e >> 1) * HALF];
      new_page = A.table[at.b * A.table_ld + (at.len - 1) / A.pool.page_size];
    }
  };
  float cs[IN][2], sn[IN][2], cs_lo[IN][2], sn_lo[IN][2];  // cosines and sines, and what f32 leaves of them
#pragma unroll
  for (int k = 0; k < IN; ++k) cs[k][0] = cs[k][1] = 1.f, sn[k][0] = sn[k][1] = 0.f;
  int64_t turned = -1;  // the sequence that cs, sn are for
  int64_t pend_row[2];  // pairs shared with other CTAs, joined at the run's end: where their output goes,
  int pend_c0[2], pend_c1[2], pend_head[2], pends = 0;  // their first and last CTA, their first query head

  int it = 0;
  bool live = true;
  if (more) load_q(W);
  while (more) {
      const int n = W.j1() - W.j0(), jb = W.j0();
      const bool has_new = A.rope && W.j1() == W.nt;
      const int64_t bh = W.b * hkv + W.hk;
      // ---- q of this set's heads: turned, scaled, as fragments ----
      if (A.rope && turned != W.b) {
#pragma unroll
        for (int k = 0; k < IN; ++k)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            double co, si;
            rope_turn(pos, rope_freq(qi + 64 * k + e, HALF, A.log2_theta), co, si);
            cs[k][e] = (float)co;
            sn[k][e] = (float)si;
            cs_lo[k][e] = (float)(co - (double)cs[k][e]);
            sn_lo[k][e] = (float)(si - (double)sn[k][e]);
          }
        turned = W.b;
      }
#pragma unroll
      for (int h = 0; h < HEADS; ++h) {
        float x[IN][4], mx = 0.f;
#pragma unroll
        for (int k = 0; k < IN; ++k)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float u = qr[h][k][e] * P.scale, y = qr[h][k][e + 2] * P.scale;
            x[k][e] = u * cs[k][e] - y * sn[k][e];
            x[k][e + 2] = u * sn[k][e] + y * cs[k][e];
            mx = fmaxf(mx, fmaxf(fabsf(x[k][e]), fabsf(x[k][e + 2])));
          }
        // a power of two that puts the head's largest |q| in [2^14, 2^15)
#pragma unroll
        for (int off = HD == 64 ? 8 : 16; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
        int ex = 0;
        if (mx > 0.f && mx <= 3.4e38f) ex = (int)((__float_as_uint(mx) >> 23) & 0xff) - 127 - 14;
        ex = max(-126, min(126, ex));
        if (qi == 0) xs_s[qh + h] = __uint_as_float((uint32_t)(127 + ex) << 23);
        const float inv = __uint_as_float((uint32_t)(127 - ex) << 23);
#pragma unroll
        for (int k = 0; k < IN; ++k)
#pragma unroll
          for (int e = 0; e < 4; e += 2) {
            const int d = qi + 64 * k + (e >> 1) * HALF;  // even: one register of a fragment
            uint32_t hi, lo;
            pa_split(x[k][e] * inv, x[k][e + 1] * inv, hi, lo);
            uint32_t* to = qf + ((d >> 4) * 32 + (qh + h) * 4 + ((d & 7) >> 1)) * 4 + ((d >> 3) & 1);
            to[0] = hi;
            to[2] = lo;
          }
      }
      if (has_new && w < 2 && (HD > 64 || lane < 16)) {
        const int64_t slot = W.len - 1;
        __half* cache = nullptr;
        if (set == 0) {
          const int64_t at = kv_row(A.pool, new_page, slot, W.hk);
          if (at >= 0) cache = static_cast<__half*>(w ? A.pool.v : A.pool.k) + at;
          if (w == 0 && lane == 0 && A.slot_pos) A.slot_pos[bh * A.track_ld + slot] = pos;
        }
#pragma unroll
        for (int k = 0; k < IN; ++k) {
          const int i = qi + 64 * k;
          __half2 a, b;
          if (w == 0) {
            float ab[2][2];
#pragma unroll
            for (int e = 0; e < 2; ++e)
              turn_key(nr[k][e], nr[k][e + 2], cs[k][e], cs_lo[k][e], sn[k][e], sn_lo[k][e], ab[0][e], ab[1][e]);
            a = __floats2half2_rn(ab[0][0], ab[0][1]);
            b = __floats2half2_rn(ab[1][0], ab[1][1]);
          } else {
            a = __floats2half2_rn(nr[k][0], nr[k][1]);
            b = __floats2half2_rn(nr[k][2], nr[k][3]);
          }
          *reinterpret_cast<__half2*>(new_s + w * HD + i) = a;
          *reinterpret_cast<__half2*>(new_s + w * HD + i + HALF) = b;
          if (cache) {
            *reinterpret_cast<__half2*>(cache + i) = a;
            *reinterpret_cast<__half2*>(cache + i + HALF) = b;
          }
        }
      }
      bar_set(set);  // (the last pair's readers of these arrays are past its joining barriers)
      const float xs0 = xs_s[2 * c], xs1 = xs_s[2 * c + 1];
      PaWalk N = W;
      more = N.next(A) && N.settle(A);
      if (more) load_q(N);  // lands while this pair is computed

      float o[C::KS][4];  // O^T: dims 16 mt + g (+ 8), heads 2c, 2c + 1
#pragma unroll
      for (int mt = 0; mt < C::KS; ++mt) o[mt][0] = o[mt][1] = o[mt][2] = o[mt][3] = 0.f;
      // heads 2c, 2c + 1; the maxima less PA_SHIFT (never -inf: slots of -inf weigh 0 next to it)
      float m0 = -FLT_MAX, m1 = -FLT_MAX, l0 = 0.f, l1 = 0.f;

      for (int t = 0; t < n; ++t, ++it) {
        const int s = it % C::STAGES;
        if (live) live = __all_sync(0xffffffffu, mbar_wait(full + s, (it / C::STAGES) & 1, A.err, KV_ERR_WAIT));
        const int64_t slot0 = (int64_t)(jb + t) * PA_TILE + 16 * w;  // this warp's first slot
        const int rows = (int)max((int64_t)0, min((int64_t)16, W.len - slot0));
        if (rows > 0 && live) {
          const uint32_t kt = ring + s * C::STAGE, vt = kt + C::TILE_B;
          if (has_new && W.len - 1 - slot0 < 16) {  // the appended row replaces what the copy found there
            const int r = (int)(W.len - 1 - slot0);
            for (int e = lane; e < 2 * (HD / 8); e += 32) {
              const int kv = e / (HD / 8), ch = e - kv * (HD / 8);
              uint8_t* dst = sm + group_off + s * C::STAGE + kv * C::TILE_B + (ch >> 3) * box_b + r * 128 +
                             (((ch & 7) ^ (r & 7)) << 4);
              *reinterpret_cast<uint4*>(dst) = reinterpret_cast<const uint4*>(new_s + kv * HD)[ch];
            }
            __syncwarp();
          }
          // S^T = K q^T: slots g, g + 8; heads 2c, 2c + 1
          float sa[2][4], sb[2][4];  // two chains each of q's parts
#pragma unroll
          for (int kk = 0; kk < C::KS; ++kk) {
            uint32_t a[4];
            pa_ldm((kt + k_lane + (kk >> 2) * box_b) ^ ((kk & 3) << 5), a);
            const uint4 f = reinterpret_cast<const uint4*>(qf)[kk * 32 + lane];
            if (kk < 2) {
              pa_mma0(sa[kk], a, f.x, f.y);
              pa_mma0(sb[kk], a, f.z, f.w);
            } else {
              pa_mma(sa[kk & 1], a, f.x, f.y);
              pa_mma(sb[kk & 1], a, f.z, f.w);
            }
          }
          // An infinite key element meets q's second parts with either sign or as 0: the first
          // parts decide (by select: 32 x 2049 slots of 128 / 8 heads take 75.3 us, with a branch 77.0)
          auto sum = [&](int i) {
            const float first = sa[0][i] + sa[1][i];
            return isinf(first) ? first : first + (sb[0][i] + sb[1][i]);
          };
          float s00 = sum(0) * xs0, s01 = sum(1) * xs1, s10 = sum(2) * xs0, s11 = sum(3) * xs1;
          if (A.mass && h0 + 2 * c < P.gp) {
            float* sp = scores + (bh * A.track_ld + slot0) * P.gp + h0 + 2 * c;
            if (g < rows) *reinterpret_cast<float2*>(sp + (int64_t)g * P.gp) = make_float2(s00, s01);
            if (g + 8 < rows) *reinterpret_cast<float2*>(sp + (int64_t)(g + 8) * P.gp) = make_float2(s10, s11);
          }
          if (rows < 16) {  // nothing behind the sequence counts, whatever lies there
            if (g >= rows) s00 = s01 = -INFINITY;
            if (g + 8 >= rows) s10 = s11 = -INFINITY;
            uint8_t* v0 = sm + group_off + s * C::STAGE + C::TILE_B;
            for (int e = lane; e < (16 - rows) * (HD / 8); e += 32) {
              const int r = rows + e / (HD / 8), ch = e % (HD / 8);
              *reinterpret_cast<uint4*>(v0 + (ch >> 3) * box_b + r * 128 + ((ch & 7) << 4)) = make_uint4(0, 0, 0, 0);
            }
            __syncwarp();
          }
          float x0 = fmaxf(s00, s10), x1 = fmaxf(s01, s11);
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) {
            x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, off));
            x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, off));
          }
          x0 = fmaxf(m0, x0 - PA_SHIFT);
          x1 = fmaxf(m1, x1 - PA_SHIFT);
          if (__any_sync(0xffffffffu, x0 != m0 || x1 != m1)) {
            const float r0 = ex2(m0 - x0), r1 = ex2(m1 - x1);
            m0 = x0;
            m1 = x1;
            l0 *= r0;
            l1 *= r1;
#pragma unroll
            for (int mt = 0; mt < C::KS; ++mt) {
              o[mt][0] *= r0;
              o[mt][1] *= r1;
              o[mt][2] *= r0;
              o[mt][3] *= r1;
            }
          }
          s00 = ex2(s00 - m0);
          s01 = ex2(s01 - m1);
          s10 = ex2(s10 - m0);
          s11 = ex2(s11 - m1);
          l0 += s00 + s10;
          l1 += s01 + s11;
          uint32_t ph0, pl0, ph1, pl1;  // P^T: slots 2c, 2c + 1 (+ 8) of head g
          pa_split(s00, s01, ph0, pl0);
          pa_split(s10, s11, ph1, pl1);
          ph0 = pa_turn(ph0);
          pl0 = pa_turn(pl0);
          ph1 = pa_turn(ph1);
          pl1 = pa_turn(pl1);
          // O^T += V^T P^T: the tile's product by itself, then a rounded add (the tensor
          // cores cut off what they add to: over a long context that would be a bias)
          auto pv = [&](float (&to)[4], const uint32_t (&a)[4]) {
            float x[4];
            pa_mma0(x, a, pl0, pl1);
            pa_mma(x, a, ph0, ph1);
#pragma unroll
            for (int k = 0; k < 4; ++k) to[k] += x[k];
          };
          const uint32_t va = vt + v_lane;
#pragma unroll
          for (int mt = 0; mt < C::KS; ++mt) {
            uint32_t a[4];
            pa_ldm_t((va + (mt >> 2) * box_b) ^ ((mt & 3) << 5), a);
            pv(o[mt], a);
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(empty + s);
      }

      // ---- the four warps' parts of the pair joined ----
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, off);
        l1 += __shfl_xor_sync(0xffffffffu, l1, off);
      }
      if (g == 0) {
        ml_s[w * 8 + 2 * c] = make_float2(m0, l0);
        ml_s[w * 8 + 2 * c + 1] = make_float2(m1, l1);
      }
      bar_set(set);
      float M0 = -INFINITY, M1 = -INFINITY, L0 = 0.f, L1 = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        M0 = fmaxf(M0, ml_s[k * 8 + 2 * c].x);
        M1 = fmaxf(M1, ml_s[k * 8 + 2 * c + 1].x);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 a = ml_s[k * 8 + 2 * c], b = ml_s[k * 8 + 2 * c + 1];
        L0 += a.y * ex2(a.x - M0);
        L1 += b.y * ex2(b.x - M1);
      }
      const float r0 = ex2(m0 - M0), r1 = ex2(m1 - M1);
#pragma unroll
      for (int mt = 0; mt < C::KS; ++mt) {
        o[mt][0] *= r0;
        o[mt][1] *= r1;
        o[mt][2] *= r0;
        o[mt][3] *= r1;
      }
      // warps 2 and 3 hand their sums to 0 and 1, then 1 to 0; a lane's own values lie 32 apart
      auto put = [&](float* to) {
#pragma unroll
        for (int mt = 0; mt < C::KS; ++mt)
#pragma unroll
          for (int k = 0; k < 4; ++k) to[(4 * mt + k) * 32 + lane] = o[mt][k];
      };
      auto add = [&](const float* from) {
#pragma unroll
        for (int mt = 0; mt < C::KS; ++mt)
#pragma unroll
          for (int k = 0; k < 4; ++k) o[mt][k] += from[(4 * mt + k) * 32 + lane];
      };
#pragma unroll 1
      for (int from = 2; from > 0; from >>= 1) {  // (one copy of the code: what is not fetched costs nothing)
        if (w >= from && w < 2 * from) put(red + (w & 1) * 8 * HD);
        bar_set(set);
        if (w < from) add(red + (from == 2 ? w : 1) * 8 * HD);
      }

      const int64_t out_row = W.b * A.out_ld + (int64_t)(W.hk * P.G + h0) * HD;
      const int head0 = (int)(W.hk * P.G + h0);
      if (n == W.nt) {
        if (w == 0) {
          const float i0 = 1.f / L0, i1 = 1.f / L1;
          float* out = A.out + out_row + 2 * c * HD + g;
#pragma unroll
          for (int mt = 0; mt < C::KS; ++mt) {
            if (2 * c < nh) {
              out[16 * mt] = o[mt][0] * i0;
              out[16 * mt + 8] = o[mt][2] * i0;
            }
            if (2 * c + 1 < nh) {
              out[HD + 16 * mt] = o[mt][1] * i1;
              out[HD + 16 * mt + 8] = o[mt][3] * i1;
            }
          }
          if (A.mass && g == 0) {
            float2* st = stats + W.b * A.hq + head0;
            if (2 * c < nh) st[2 * c] = make_float2(M0, L0);
            if (2 * c + 1 < nh) st[2 * c + 1] = make_float2(M1, L1);
          }
        }
      } else {
        const int c0 = W.c0();
        if (w == 0) {
          const int64_t at = ((2 * (int64_t)blockIdx.x + ((int)blockIdx.x == c0)) * NS + set) * 8;
          float* to = part + at * HD + 2 * c * HD + g;
#pragma unroll
          for (int mt = 0; mt < C::KS; ++mt) {
            to[16 * mt] = o[mt][0];
            to[16 * mt + 8] = o[mt][2];
            to[HD + 16 * mt] = o[mt][1];
            to[HD + 16 * mt + 8] = o[mt][3];
          }
          if (g == 0) {
            part_ml[at + 2 * c] = make_float2(M0, L0);
            part_ml[at + 2 * c + 1] = make_float2(M1, L1);
          }
        }
        // only a run's first and last pair can be shared: at most two
        const int k = pends++;
        pend_row[k & 1] = out_row;
        pend_head[k & 1] = (int)(W.b * A.hq) + head0;
        pend_c0[k & 1] = c0;
        pend_c1[k & 1] = W.c1();
      }
      W = N;
  }
  if (!pends) return;

  // ---- shared pairs: the last CTA to arrive joins the parts in slot order ----
  if (NS > 1) asm volatile("bar.sync 3, %0;" ::"n"(C::CW * 32) : "memory");  // the ring is used up by every set
  if (w == 0) {
    __syncwarp();
    if (lane < pends) {
      __threadfence();  // the warp's parts before the arrival, and what the arrival found before the join
      unsigned* cnt = ctr + 2 * (lane ? pend_c0[1] : pend_c0[0]) + set;
      const int others = lane ? pend_c1[1] - pend_c0[1] : pend_c1[0] - pend_c0[0];
      const bool last = atomicAdd(cnt, 1u) == (unsigned)others;
      if (last) {
        __threadfence();
        *cnt = 0u;  // ready for the next call (stream-ordered)
      }
      last_s[lane] = last;
    }
  }
  bar_set(set);
  for (int k = 0; k < pends; ++k) {
    if (!last_s[k]) continue;
    const int c0 = k ? pend_c0[1] : pend_c0[0], parts = (k ? pend_c1[1] : pend_c1[0]) - c0 + 1;
    const int64_t out_row = k ? pend_row[1] : pend_row[0];
    const int head0 = k ? pend_head[1] : pend_head[0];
    // part p's place: the pair begins in c0's second slot and goes on in the others' first
    auto place = [&](int p) { return ((2 * (int64_t)(c0 + p) + (p == 0)) * NS + set) * 8; };
    // every part's {max, sum} into the ring (its copies are used up); while they
    // come, the first sums: a thread takes a float4 column of parts pg, pg + np, ...
    const int cols = nh * (HD / 4), np = max(1, PA_SET / cols);
    float2* ml_p = reinterpret_cast<float2*>(sm) + set * C::PARTS * 8;
    for (int e = stid; e < parts * nh; e += PA_SET) ml_p[e] = __ldcg(part_ml + place(e / nh) + e % nh);
    constexpr int AHEAD = 8;  // (16 took 1.8 us more of 54 at 32 sequences of 2049: a longer kernel)
    for (int e = stid; e < (np > 1 ? PA_SET : (cols + PA_SET - 1) / PA_SET * PA_SET); e += PA_SET) {
      const int pg = np > 1 ? e / cols : 0, col = np > 1 ? e - pg * cols : e;
      const bool mine = pg < np && col < cols;
      const int h = mine ? col / (HD / 4) : 0, d4 = col - h * (HD / 4);
      auto sum_of = [&](int p) {
        return mine && p < parts ? __ldcg(reinterpret_cast<const float4*>(part + (place(p) + h) * HD) + d4)
                                 : make_float4(0.f, 0.f, 0.f, 0.f);
      };
      float4 v[AHEAD];
#pragma unroll
      for (int q = 0; q < AHEAD; ++q) v[q] = sum_of(pg + q * np);
      bar_set(set);
      float M = -INFINITY, L = 0.f;
      for (int p = 0; p < parts; ++p) M = fmaxf(M, ml_p[p * nh + h].x);
      float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int p0 = pg; p0 < parts; p0 += AHEAD * np) {
#pragma unroll
        for (int q = 0; q < AHEAD; ++q) {
          const int p = p0 + q * np;
          const float2 ml = p < parts ? ml_p[p * nh + h] : make_float2(-INFINITY, 0.f);
          const float f = ex2(ml.x - M);
          L = fmaf(f, ml.y, L);
          r.x = fmaf(f, v[q].x, r.x);
          r.y = fmaf(f, v[q].y, r.y);
          r.z = fmaf(f, v[q].z, r.z);
          r.w = fmaf(f, v[q].w, r.w);
          v[q] = sum_of(p + AHEAD * np);
        }
      }
      if (np > 1) {  // the parts' groups, in order
        float4* rs = reinterpret_cast<float4*>(red);
        rs[stid] = r;
        float* ls = red + PA_SET * 4;
        ls[stid] = L;
        bar_set(set);
        if (pg == 0) {
          for (int q = 1; q < np; ++q) {
            const float4 x = rs[q * cols + col];
            r.x += x.x;
            r.y += x.y;
            r.z += x.z;
            r.w += x.w;
            L += ls[q * cols + col];
          }
        }
      }
      if (mine && pg == 0) {
        const float inv = 1.f / L;
        float* out = A.out + out_row + h * HD + 4 * d4;
        out[0] = r.x * inv;
        out[1] = r.y * inv;
        out[2] = r.z * inv;
        out[3] = r.w * inv;
        if (A.mass && d4 == 0) stats[head0 + h] = make_float2(M, L);
      }
    }
    bar_set(set);  // ml_p and red are free again
  }
}

// mass[slot] += sum over the group's heads of 2^(s - M) / L, from the scores and
// the joined maxima and sums of the kernel above.
__global__ void __launch_bounds__(256) kv_mass_kernel(const __grid_constant__ PaParams P) {
  kv_pdl_enter();
  const KvAttnArgs& A = P.a;
  __shared__ float2 stats[KV_MAX_GROUP];  // {max, 1 / sum}
  const int hk = blockIdx.y;
  const int64_t b = blockIdx.z, bh = b * A.pool.hkv + hk;
  const char* scratch = static_cast<const char*>(A.scratch);
  if (threadIdx.x < P.G) {
    const float2 ml = (reinterpret_cast<const float2*>(scratch + P.at.stats) + b * A.hq + hk * P.G)[threadIdx.x];
    stats[threadIdx.x] = make_float2(ml.x, 1.f / ml.y);
  }
  bool bad;
  const int len = pa_len(A, b, &bad);
  __syncthreads();
  const float2* scores = reinterpret_cast<const float2*>(scratch + P.at.scores) + bh * A.track_ld * (P.gp / 2);
  float* mass = A.mass + bh * A.track_ld;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < len; i += (int64_t)gridDim.x * blockDim.x) {
    const float old = A.rope && i == len - 1 ? 0.f : mass[i];
    float v = 0.f;
#pragma unroll 4
    for (int h = 0; h < P.G; h += 2) {
      const float2 s = scores[i * (P.gp / 2) + h / 2];
      v += ex2(s.x - stats[h].x) * stats[h].y;
      if (h + 1 < P.G) v += ex2(s.y - stats[h + 1].x) * stats[h + 1].y;
    }
    mass[i] = old + v;
  }
}

template <int HD, int NS>
cudaError_t launch_attn(const PaParams& P, const KvMaps& maps, int num_sms, cudaStream_t s) {
  using C = PaCfg<HD, NS>;
  const KvAttnArgs& a = P.a;
  const int64_t tiles = a.batch * a.pool.hkv * ((a.table_cols * a.pool.page_size + PA_TILE - 1) / PA_TILE);
  const unsigned grid = (unsigned)std::min<int64_t>(std::min<int64_t>(C::CTAS * num_sms, C::PARTS), tiles);
  return launch_pdl(kv_attn_kernel<HD, NS>, dim3(grid), dim3(C::THREADS), C::END, s, maps.k, maps.v, P);
}

template <int HD>
cudaError_t launch_attn_hd(const PaParams& P, const KvMaps& maps, int num_sms, cudaStream_t s) {
  return P.G <= 8 ? launch_attn<HD, 1>(P, maps, num_sms, s) : launch_attn<HD, 2>(P, maps, num_sms, s);
}

template <int HD, int NS>
cudaError_t attn_attr() {
  return cudaFuncSetAttribute(kv_attn_kernel<HD, NS>, cudaFuncAttributeMaxDynamicSharedMemorySize, PaCfg<HD, NS>::END);
}

}  // namespace

bool kv_make_maps(const KvPool& p, KvMaps* maps) {
  // innermost first: 64 dims, the page's slots, the 64-dim halves of a row, heads, pages
  const cuuint64_t dims[5] = {64, (cuuint64_t)p.page_size, (cuuint64_t)p.hd / 64, (cuuint64_t)p.hkv,
                              (cuuint64_t)p.pages};
  const cuuint64_t strides[4] = {(cuuint64_t)p.hd * 2, 128, (cuuint64_t)p.page_size * p.hd * 2,
                                 (cuuint64_t)p.page_ld * 2};
  const cuuint32_t box[5] = {64, (cuuint32_t)kv_box_rows(p.page_size), (cuuint32_t)p.hd / 64, 1, 1};
  return encode_tiled_map(&maps->k, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 5, p.k, dims, strides, box,
                          CU_TENSOR_MAP_SWIZZLE_128B) &&
         encode_tiled_map(&maps->v, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 5, p.v, dims, strides, box,
                          CU_TENSOR_MAP_SWIZZLE_128B);
}

cudaError_t kv_init_device() {
  cudaError_t e = attn_attr<64, 1>();
  if (e == cudaSuccess) e = attn_attr<64, 2>();
  if (e == cudaSuccess) e = attn_attr<128, 1>();
  if (e == cudaSuccess) e = attn_attr<128, 2>();
  if (e == cudaSuccess) e = attn_attr<256, 1>();
  if (e == cudaSuccess) e = attn_attr<256, 2>();
  return e;
}

size_t kv_attention_scratch_bytes(int64_t batch, int hq, int hkv, int hd, int64_t track_len, int num_sms) {
  // the scores alone; the rest is far below 2^60
  if (kv_too_many(batch * hkv, track_len, (hq / hkv + 1) * (int64_t)sizeof(float))) return SIZE_MAX;
  return PaScratch(batch, hq, hkv, hd, track_len, num_sms).end;
}

cudaError_t kv_attention(const KvAttnArgs& a, const KvMaps& maps, int* launches, cudaStream_t s) {
  PaParams P{a, PaScratch(a.batch, a.hq, a.pool.hkv, a.pool.hd, a.mass ? a.track_ld : 0, a.num_sms)};
  P.G = a.hq / a.pool.hkv;
  P.gp = (P.G + 1) & ~1;
  P.box = kv_box_rows(a.pool.page_size);
  P.scale = (float)(1.4426950408889634 / sqrt((double)a.pool.hd));
  cudaError_t e = a.pool.hd == 64    ? launch_attn_hd<64>(P, maps, a.num_sms, s)
                  : a.pool.hd == 128 ? launch_attn_hd<128>(P, maps, a.num_sms, s)
                                     : launch_attn_hd<256>(P, maps, a.num_sms, s);
  if (e != cudaSuccess) return e;
  *launches = 1;
  if (!a.mass) return e;
  const int64_t most = std::min(a.track_ld, a.table_cols * a.pool.page_size);
  const unsigned chunks = (unsigned)std::min<int64_t>((most + 511) / 512, 64);
  e = launch_pdl(kv_mass_kernel, dim3(chunks, (unsigned)a.pool.hkv, (unsigned)a.batch), dim3(256), 0, s, P);
  *launches += e == cudaSuccess;
  return e;
}

}  // namespace kq
