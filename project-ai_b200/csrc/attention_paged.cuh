// What the paged attention kernels share: their arguments and the reading of a request's row range and length.
#pragma once

#include <math.h>

#include "paged.cuh"

namespace pai {
namespace paged {

struct AttnArgs {
  const float* q; int64_t q0, q1;          // row, head strides
  const float* k;
  const float* v;
  int64_t c0, c1, c2;                      // page, head, position strides of both caches
  const float* table; int64_t t0, t1;
  const float* start; int64_t start_s;     // q_start [n + 1]
  const float* len; int64_t len_s;         // kv_len [n]
  float* out;                              // [rows, H, D]
  int n, rows, H, KVH, g, D, max_pages, pages, max_new;
  PageDiv page, heads;                     // division by the page size, by g
  // scale * log2(e), so that scores are powers of two, in two parts: q hi + q lo is off by one rounding (a scale in one
  // part would bend all scores alike, by up to 2^-24 of themselves)
  float scale_hi, scale_lo;
  int vec, q_vec;                          // cache rows, rows of q may be read as float4
  int whole_groups;                        // ... and no group of keys straddles pages
  float* part;                             // partial results, two slots per block
  unsigned* tickets;                       // arrivals, one counter per block (all zero between launches)
  int* error_flag;
};

struct Req {
  int first, n, len;  // first row, new tokens, keys
  bool placed;        // its row range is valid
};

// Request i; false when its values are invalid (sets the error flag), n = 0 when it has no new token.
__device__ __forceinline__ bool load_req(const AttnArgs& a, int i, Req& r) {
  const float first = a.start[i * a.start_s], last = a.start[(i + 1) * a.start_s], keys = a.len[i * a.len_s];
  int end = 0;
  r.first = r.n = r.len = 0;
  r.placed = integral(first, 0, a.rows, r.first) && integral(last, 0, a.rows, end) && end >= r.first;
  if (!r.placed || !integral(keys, 0, a.max_pages * a.page.size, r.len) || end - r.first > a.max_new) return false;
  r.n = end - r.first;
  return true;
}

// Rows of out that belong to no request are zero: those before the first request and behind the last, when all row ranges
// are valid (else a row behind the last range may be another request's).
__device__ __forceinline__ void zero_rest(const AttnArgs& a) {
  const float first = a.start[0], last = a.start[a.n * a.start_s];
  int lo, hi;
  if (!integral(first, 0, a.rows, lo) || !integral(last, 0, a.rows, hi)) return;
  const int per = a.H * a.D, rest = lo + (a.rows - hi);
#pragma unroll 1
  for (int r = blockIdx.x; r < rest; r += gridDim.x) {
    float* o = a.out + (int64_t)(r < lo ? r : hi + (r - lo)) * per;
#pragma unroll 1
    for (int e = threadIdx.x; e < per; e += blockDim.x) o[e] = 0.0f;
  }
}

// The tensor-core kernel (attention_paged_tc.cu): whether it takes this call, the device memory for its partial
// results, and its launch.
bool tc_fits(const AttnArgs& a);
size_t tc_part_bytes(const pai_ctx* ctx);
pai_status tc_launch(pai_ctx* ctx, const AttnArgs& a);

}  // namespace paged
}  // namespace pai
