// Argument checks of the paged KV cache entry points (pai_paged_plan, pai_paged_rope_append, pai_sdpa_paged): plain
// host code on the view descriptors, compiled into the CUDA library and into the CPU oracle alike, so both refuse the
// same calls with the same messages.
#pragma once

#include <stdint.h>

#include "projectai_cuda.h"

namespace pai_paged {

typedef pai_status (*Fail)(pai_status, const char*, ...);

// F32 holds every integer up to 2^24: the bound on slots, positions and rows.
constexpr int64_t kMaxIndex = 1 << 24;
constexpr int kMaxHeadDim = 128;
// rows x heads of one attention call, and its requests: the kernels count them, rounded up to their tiles, in 32 bits.
constexpr int64_t kMaxQueryRows = 1 << 30;

// An in-place operand: no two elements at one address by a zero stride.
inline bool writable(const pai_tensor& t) {
  for (int i = 0; i < t.rank; i++)
    if (t.dims[i] > 1 && t.strides[i] == 0) return false;
  return true;
}

// Whether two views have an element in common: whether sum i_k s_k - sum j_k t_k = the distance of their first elements has a
// solution within their dims. The terms are tried from the widest on, as far as those left can reach the rest, which for
// nested and interleaved layouts are one or two at each; views whose search takes longer count as apart.
class Overlap {
  int64_t coef_[2 * PAI_MAX_RANK], most_[2 * PAI_MAX_RANK], reach_[2 * PAI_MAX_RANK + 1];
  int terms_ = 0, budget_ = 4096;
  bool search(int k, int64_t rest) {
    if (rest < 0 || rest > reach_[k]) return false;
    if (k == terms_) return rest == 0;
    const int64_t hi = rest / coef_[k] < most_[k] ? rest / coef_[k] : most_[k];
    const int64_t need = rest - reach_[k + 1];
    for (int64_t i = need > 0 ? (need + coef_[k] - 1) / coef_[k] : 0; i <= hi; i++) {
      if (budget_-- <= 0) return false;
      if (search(k + 1, rest - i * coef_[k])) return true;
    }
    return false;
  }
  bool add(const pai_tensor& t, int64_t sign, int64_t* rest) {  // false: the view is empty
    for (int i = 0; i < t.rank; i++) {
      if (t.dims[i] == 0) return false;
      int64_t c = sign * t.strides[i];
      const int64_t n = t.dims[i] - 1;
      if (n == 0 || c == 0) continue;
      if (c < 0) {  // counted from the other end
        *rest -= c * n;
        c = -c;
      }
      int at = 0;
      while (at < terms_ && coef_[at] > c) at++;
      if (at < terms_ && coef_[at] == c) {
        most_[at] += n;
        continue;
      }
      for (int k = terms_++; k > at; k--) {
        coef_[k] = coef_[k - 1];
        most_[k] = most_[k - 1];
      }
      coef_[at] = c;
      most_[at] = n;
    }
    return true;
  }

  static bool in_one_block(const pai_tensor& a, const pai_tensor& b) {
    Overlap o;
    int64_t rest = b.offset - a.offset;
    if (!o.add(a, 1, &rest) || !o.add(b, -1, &rest)) return false;
    o.reach_[o.terms_] = 0;
    for (int k = o.terms_ - 1; k >= 0; k--) o.reach_[k] = o.reach_[k + 1] + o.coef_[k] * o.most_[k];
    return o.search(0, rest);
  }

 public:
  static bool of(const pai_tensor& a, const pai_tensor& b) { return a.base == b.base && in_one_block(a, b); }
};

inline pai_status check_plan(Fail fail, const pai_tensor* lengths, const pai_tensor* new_tokens, const pai_tensor* table,
                             const pai_tensor* ring, const pai_tensor* state, int32_t page_size, int32_t rows) {
  if (lengths->rank != 1 || new_tokens->rank != 1 || table->rank != 2 || ring->rank != 1 || state->rank != 1 ||
      state->dims[0] != 2)
    return fail(PAI_ERR_ARGUMENT, "PagedPlan: lengths [N], new_tokens [N], table [N, max_pages], ring [pages] and state [2] expected");
  const int n = lengths->dims[0];
  if (new_tokens->dims[0] != n || table->dims[0] != n)
    return fail(PAI_ERR_ARGUMENT, "PagedPlan: %d lengths, %d new_tokens and %d rows of table disagree", n,
                new_tokens->dims[0], table->dims[0]);
  if (page_size < 1) return fail(PAI_ERR_OUT_OF_RANGE, "PagedPlan: page size %d", page_size);
  if (rows < 0) return fail(PAI_ERR_OUT_OF_RANGE, "PagedPlan: %d rows", rows);
  if (rows > kMaxIndex || (int64_t)ring->dims[0] * page_size > kMaxIndex || (int64_t)table->dims[1] * page_size > kMaxIndex)
    return fail(PAI_ERR_UNSUPPORTED, "PagedPlan: %d rows, %d pages of %d positions, %d pages per request: above 2^24, F32 holds no exact ids",
                rows, ring->dims[0], page_size, table->dims[1]);
  if (!writable(*table) || !writable(*ring))
    return fail(PAI_ERR_ARGUMENT, "PagedPlan: table and ring are written in place and cannot be broadcast views");
  const pai_tensor* all[5] = {lengths, new_tokens, table, ring, state};
  for (int w = 2; w < 4; w++)
    for (int i = 0; i < 5; i++)
      if (i != w && Overlap::of(*all[i], *all[w]))
        return fail(PAI_ERR_ARGUMENT, "PagedPlan: table and ring are written in place and cannot share elements with another operand");
  return PAI_OK;
}

// Both caches [pages, KVH, P, D] of one layout.
inline pai_status check_caches(Fail fail, const char* op, const pai_tensor* k_cache, const pai_tensor* v_cache) {
  if (k_cache->rank != 4 || v_cache->rank != 4)
    return fail(PAI_ERR_ARGUMENT, "%s: caches [pages, KVH, P, D] expected", op);
  for (int i = 0; i < 4; i++)
    if (k_cache->dims[i] != v_cache->dims[i] || (k_cache->dims[i] > 1 && k_cache->strides[i] != v_cache->strides[i]))
      return fail(PAI_ERR_ARGUMENT, "%s: k and v caches must share one layout", op);
  if (k_cache->dims[1] < 1 || k_cache->dims[2] < 1 || k_cache->dims[3] < 1)
    return fail(PAI_ERR_ARGUMENT, "%s: caches with an empty page", op);
  if (k_cache->dims[3] > 1 && k_cache->strides[3] != 1)
    return fail(PAI_ERR_UNSUPPORTED, "%s: the caches' head dim must be contiguous", op);
  if ((int64_t)k_cache->dims[0] * k_cache->dims[2] > kMaxIndex)
    return fail(PAI_ERR_UNSUPPORTED, "%s: %d pages of %d positions: above 2^24, F32 holds no exact slots", op,
                k_cache->dims[0], k_cache->dims[2]);
  return PAI_OK;
}

inline pai_status check_append(Fail fail, const pai_tensor* q, const pai_tensor* k, const pai_tensor* v,
                               const pai_tensor* cos_table, const pai_tensor* sin_table, const pai_tensor* positions,
                               const pai_tensor* slots, const pai_tensor* k_cache, const pai_tensor* v_cache) {
  if (q->rank != 3 || k->rank != 3 || v->rank != 3 || cos_table->rank != 2 || sin_table->rank != 2 || positions->rank != 1 ||
      slots->rank != 1)
    return fail(PAI_ERR_ARGUMENT, "PagedRopeAppend: q [rows,H,D], k and v [rows,KVH,D], [T,D] tables, positions and slots [rows] expected");
  const pai_status st = check_caches(fail, "PagedRopeAppend", k_cache, v_cache);
  if (st != PAI_OK) return st;
  const int rows = q->dims[0], d = q->dims[2];
  for (int i = 0; i < 3; i++)
    if (k->dims[i] != v->dims[i]) return fail(PAI_ERR_ARGUMENT, "PagedRopeAppend: k and v shapes differ");
  if (k->dims[0] != rows || positions->dims[0] != rows || slots->dims[0] != rows)
    return fail(PAI_ERR_ARGUMENT, "PagedRopeAppend: %d rows of q, %d of k, %d positions and %d slots disagree", rows,
                k->dims[0], positions->dims[0], slots->dims[0]);
  if (k->dims[2] != d || k_cache->dims[1] != k->dims[1] || k_cache->dims[3] != d)
    return fail(PAI_ERR_ARGUMENT, "PagedRopeAppend: q, k and the caches disagree on heads or head dim");
  if (d % 2) return fail(PAI_ERR_ARGUMENT, "PagedRopeAppend: odd head dim %d", d);
  if (cos_table->dims[1] != d || sin_table->dims[1] != d || sin_table->dims[0] != cos_table->dims[0])
    return fail(PAI_ERR_ARGUMENT, "PagedRopeAppend: tables must be [T, %d]", d);
  // a longer table's last row would round up to one behind it where positions are compared with it
  if (cos_table->dims[0] > kMaxIndex)
    return fail(PAI_ERR_UNSUPPORTED, "PagedRopeAppend: tables of %d rows: above 2^24, F32 holds no exact positions",
                cos_table->dims[0]);
  if (q->strides[2] != 1 || k->strides[2] != 1 || v->strides[2] != 1 || cos_table->strides[1] != 1 ||
      sin_table->strides[1] != 1 || (cos_table->dims[0] > 1 && cos_table->strides[0] != sin_table->strides[0]))
    return fail(PAI_ERR_UNSUPPORTED, "PagedRopeAppend: rows must be contiguous and the tables share one layout");
  if (!writable(*k_cache) || !writable(*v_cache))
    return fail(PAI_ERR_ARGUMENT, "PagedRopeAppend: the caches are written in place and cannot be broadcast views");
  const pai_tensor* others[7] = {q, k, v, cos_table, sin_table, positions, slots};
  bool shared = Overlap::of(*k_cache, *v_cache);
  for (int i = 0; i < 7; i++) shared = shared || Overlap::of(*others[i], *k_cache) || Overlap::of(*others[i], *v_cache);
  if (shared)
    return fail(PAI_ERR_ARGUMENT, "PagedRopeAppend: the caches are written in place and cannot share elements with one another or another operand");
  return PAI_OK;
}

inline pai_status check_sdpa(Fail fail, const pai_tensor* q, const pai_tensor* k_cache, const pai_tensor* v_cache,
                             const pai_tensor* table, const pai_tensor* q_start, const pai_tensor* kv_len, int32_t max_new) {
  if (q->rank != 3 || table->rank != 2 || q_start->rank != 1 || kv_len->rank != 1)
    return fail(PAI_ERR_ARGUMENT, "SdpaPaged: q [rows,H,D], table [N, max_pages], q_start [N+1] and kv_len [N] expected");
  const pai_status st = check_caches(fail, "SdpaPaged", k_cache, v_cache);
  if (st != PAI_OK) return st;
  const int n = table->dims[0], h = q->dims[1], d = q->dims[2], kvh = k_cache->dims[1];
  if (q_start->dims[0] != n + 1 || kv_len->dims[0] != n)
    return fail(PAI_ERR_ARGUMENT, "SdpaPaged: table of %d requests needs q_start [%d] and kv_len [%d], got [%d] and [%d]", n,
                n + 1, n, q_start->dims[0], kv_len->dims[0]);
  if (k_cache->dims[3] != d || h % kvh)
    return fail(PAI_ERR_ARGUMENT, "SdpaPaged: %d query heads of %d do not fit %d kv heads of %d", h, d, kvh, k_cache->dims[3]);
  if (d > kMaxHeadDim) return fail(PAI_ERR_UNSUPPORTED, "SdpaPaged: head dim %d above %d", d, kMaxHeadDim);
  if (d > 1 && q->strides[2] != 1) return fail(PAI_ERR_UNSUPPORTED, "SdpaPaged: rows of q must be contiguous along the head dim");
  if (max_new < 0) return fail(PAI_ERR_OUT_OF_RANGE, "SdpaPaged: max_new %d", max_new);
  if (q->dims[0] > kMaxIndex || (int64_t)table->dims[1] * k_cache->dims[2] > kMaxIndex)
    return fail(PAI_ERR_UNSUPPORTED, "SdpaPaged: %d rows, %d pages of %d positions per request: above 2^24, F32 holds no exact positions",
                q->dims[0], table->dims[1], k_cache->dims[2]);
  if ((int64_t)q->dims[0] * h > kMaxQueryRows || n > kMaxQueryRows)
    return fail(PAI_ERR_UNSUPPORTED, "SdpaPaged: %d rows of %d heads, %d requests: above 2^30", q->dims[0], h, n);
  return PAI_OK;
}

}  // namespace pai_paged
