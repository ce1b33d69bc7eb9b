// Addressing of a paged cache, shared by the device code and its host check.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace nsa {

// Element offset of the first row of run `run` (16 positions, all in one page)
// of one sequence and KV head, or -1 where the run has no page.  `row` is the
// sequence's table row, rpp the runs of a page (P / 16).
__host__ __device__ inline int64_t paged_run(const int32_t* row, int run, int rpp, int max_pages, int n_pages, int Hkv,
                                             int hkv, int D) {
  const int pi = run / rpp;
  if (run < 0 || pi >= max_pages) return -1;
  const int page = row[pi];
  if (page < 0 || page >= n_pages) return -1;
  return (((int64_t)page * Hkv + hkv) * rpp + (run - pi * rpp)) * 16 * D;
}

// Position of the row a step appends, or -1 where it has no page.
__host__ __device__ inline int paged_new_pos(const int32_t* row, int len, int P, int max_pages, int n_pages) {
  if (len < 0 || len >= max_pages * P) return -1;
  const int page = row[len / P];
  return page >= 0 && page < n_pages ? len : -1;
}

}  // namespace nsa
