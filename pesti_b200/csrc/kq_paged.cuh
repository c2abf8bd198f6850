// kq_paged.cuh -- addressing of the paged key-value cache and the rotary
// angle, shared by the kernels of kq_paged.cu (host-callable, so that the
// index arithmetic can be checked without a GPU).
#pragma once

#include <stdint.h>

#include "kq_kernels.h"

namespace kq {

// Device error codes of the paged cache and its callers (the context's error word).
enum : int { KV_ERR_PAGE = 51, KV_ERR_LEN = 52, KV_ERR_ROW = 53, KV_ERR_WAIT = 54 };

// A sequence's slots in use: lens[b] held to [0, most]; *bad is set where it was outside.
__host__ __device__ __forceinline__ int64_t kv_len(int32_t len, int64_t most, bool* bad) {
  *bad = len < 0 || len > most;
  return len < 0 ? 0 : len > most ? most : (int64_t)len;
}

// Element offset of slot's row for one kv head, or -1 where the table's page
// is outside the pool.
__host__ __device__ __forceinline__ int64_t kv_row(const KvPool& p, int32_t page, int64_t slot, int head) {
  if (page < 0 || page >= p.pages) return -1;
  return (int64_t)page * p.page_ld + ((int64_t)head * p.page_size + slot % p.page_size) * p.hd;
}

}  // namespace kq
