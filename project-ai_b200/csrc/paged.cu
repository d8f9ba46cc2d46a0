// Paged KV cache, the step before the attention: planning (which pages and slots the new tokens get) and the
// rotate-and-append into them. The attention that reads the pages is in attention_paged.cu.
#include "paged.cuh"

namespace pai {
namespace paged {

// ---------------------------------------------------------------- plan
// l = lengths, a = new tokens (-1: ended), P = page size:
//   have = ceil(l / P), need = ceil((l + a) / P) - have, back = have for an ended request;
//   table[i, have + r] = ring[(head + sum_{j<i} need_j + r) mod R]; the pages of ended requests go to
//   ring[(head + count + ...) mod R]; token t of request i: pos = l + t - q_start[i], slot = page(pos) * P + pos mod P.
// One launch: every block sums the requests itself (a thread sums `per` consecutive requests, a block scan joins them),
// then the grid's threads share three flat lists, the rows, the pages taken and the pages returned; the request of a
// list's element is found by bisection over the scanned sums. A token in a new page computes its id from the ring,
// not from table, so no block reads what another writes: rows of table are read below have and written from have on;
// ring is read in [head, head + taken) and written from head + count on, and count + returned <= R keeps the two apart.
// Bound by launch latency: 8 requests and 1,000 requests 3.3 us on the device.
constexpr int kPlanThreads = 256;

struct PlanArgs {
  const float* len; int64_t len_s;
  const float* add; int64_t add_s;
  float* table; int64_t t0, t1;
  float* ring; int64_t ring_s;
  const float* state; int64_t state_s;
  int n, max_pages, pages, rows, per;
  PageDiv page;
  float *q_start, *kv_len, *slots, *positions, *next_state;
  int* error_flag;
};

struct PlanReq {
  int len, add, have, need, back;
  bool ok, ended;
};

__device__ __forceinline__ PlanReq plan_req(const PlanArgs& a, int i) {
  PlanReq r{};
  const int cap = a.max_pages * a.page.size;
  r.ok = integral(a.len[i * a.len_s], 0, cap, r.len);
  if (!r.ok) r.len = 0;
  int add = 0;
  if (!integral(a.add[i * a.add_s], -1, a.rows, add)) { r.ok = false; add = 0; }
  r.ended = add < 0;
  r.add = max(add, 0);
  if (r.len > cap - r.add) { r.ok = false; r.add = 0; }
  r.have = a.page.div(r.len + a.page.size - 1);
  r.need = r.ended ? 0 : a.page.div(r.len + r.add + a.page.size - 1) - r.have;
  r.back = r.ended ? r.have : 0;
  return r;
}

__global__ void __launch_bounds__(kPlanThreads) k_paged_plan(const PlanArgs a) {
  __shared__ int pre[3][kPlanThreads + 1];  // exclusive sums of tokens, pages taken, pages returned over the threads
  __shared__ int64_t tmp[3 * kPlanThreads / 32];
  pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x, P = a.page.size;
  const int i0 = min(a.n, tid * a.per), i1 = min(a.n, i0 + a.per);
  int64_t sum[3] = {0, 0, 0};
  bool ok = true;
  for (int i = i0; i < i1; i++) {
    const PlanReq r = plan_req(a, i);
    ok = ok && r.ok;
    sum[0] += r.add;
    sum[1] += r.need;
    sum[2] += r.back;
  }
  int head = 0, count = 0;
  ok = ok && integral(a.state[0], 0, max(0, a.pages - 1), head) && integral(a.state[a.state_s], 0, a.pages, count);
  int64_t total[3], sums_before[3];
  block_prefix<kPlanThreads>(sum, tmp, sums_before, total);
#pragma unroll
  for (int k = 0; k < 3; k++) {
    pre[k][tid] = (int)min(sums_before[k], (int64_t)INT32_MAX);
    if (tid == kPlanThreads - 1) pre[k][kPlanThreads] = (int)min(total[k], (int64_t)INT32_MAX);
  }
  ok = __syncthreads_and(ok) && total[0] <= a.rows && total[1] <= count && count + total[2] <= a.pages;

  const int gsize = gridDim.x * kPlanThreads, gid = blockIdx.x * kPlanThreads + tid;
  if (blockIdx.x == 0) {
    int start = pre[0][tid];
    for (int i = i0; i < i1; i++) {
      const PlanReq r = plan_req(a, i);
      start += r.add;
      a.q_start[i + 1] = ok ? (float)start : 0.0f;
      a.kv_len[i] = ok && r.ended ? 0.0f : (float)(r.len + (ok ? r.add : 0));
    }
    if (tid == 0) {
      a.q_start[0] = 0.0f;
      int next = 0;
      if (ok && a.pages > 0) next = (int)((head + total[1]) % a.pages);
      a.next_state[0] = ok ? (float)next : a.state[0];
      a.next_state[1] = ok ? (float)(count - total[1] + total[2]) : a.state[a.state_s];
      if (!ok) atomicExch(a.error_flag, 70);
    }
  }
  // Element f of list k: the thread whose sums hold it, then its requests one by one. `need_before`: pages taken by the
  // requests before the one found.
  auto find = [&](int k, int f, PlanReq& r, int& i, int& rest, int& need_before) {
    int lo = 0, hi = kPlanThreads;  // pre[k][lo] <= f < pre[k][hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (pre[k][mid] <= f) lo = mid;
      else hi = mid;
    }
    i = lo * a.per;
    rest = f - pre[k][lo];
    need_before = pre[1][lo];
    for (;; i++) {
      r = plan_req(a, i);
      const int n = k == 0 ? r.add : k == 1 ? r.need : r.back;
      if (rest < n) return;
      rest -= n;
      need_before += r.need;
    }
  };
  PlanReq r;
  int i, rest, before;
  const int tokens = ok ? (int)total[0] : 0;
  for (int t = gid; t < a.rows; t += gsize) {
    float slot = -1.0f, pos = 0.0f;
    if (t < tokens) {
      find(0, t, r, i, rest, before);
      const int p = r.len + rest, pi = a.page.div(p);
      pos = (float)p;
      const float id = pi < r.have ? a.table[i * a.t0 + pi * a.t1]
                                   : a.ring[(int64_t)((head + before + (pi - r.have)) % a.pages) * a.ring_s];
      int page;
      if (integral(id, 0, a.pages - 1, page)) slot = (float)(page * P + (p - pi * P));
      else atomicExch(a.error_flag, 71);
    }
    a.slots[t] = slot;
    a.positions[t] = pos;
  }
  if (!ok) return;
  for (int f = gid; f < (int)total[1]; f += gsize) {
    find(1, f, r, i, rest, before);
    a.table[i * a.t0 + (int64_t)(r.have + rest) * a.t1] = a.ring[(int64_t)((head + f) % a.pages) * a.ring_s];
  }
  for (int f = gid; f < (int)total[2]; f += gsize) {
    find(2, f, r, i, rest, before);
    a.ring[(int64_t)((head + count + f) % a.pages) * a.ring_s] = a.table[i * a.t0 + rest * a.t1];
  }
}

// ---------------------------------------------------------------- rotate and append
// y[j] = x[j] cos[j] - x[j+h] sin[j], y[j+h] = x[j+h] cos[j+h] + x[j] sin[j+h] (h = D / 2), rounded as k_rope_append
// rounds it (RotaryEmbedding, CpuComputeBackend.cs:397-420). Bound by HBM: each element is read once and written once.
// A thread takes elements j.. and j+h.. (4 of each with VEC) of several heads of one row, so the row's table entries,
// position and slot are read once for them; heads are q's, then k's, then v's. 13,657 rows of 32 + 2·8 heads of 64: 61 us,
// 5.5 TB/s.
struct AppendArgs {
  const float* q; int64_t q0, q1;
  const float* k; int64_t k0, k1;
  const float* v; int64_t v0, v1;
  const float* cos;
  const float* sin;
  int64_t tab;
  const float* pos; int64_t pos_s;
  const float* slot; int64_t slot_s;
  float* kc;
  float* vc;
  int64_t c0, c1, c2;  // page, head, position strides of both caches
  float* q_out;
  int rows, H, KVH, D, tab_rows, slots;
  PageDiv page;
  int groups;  // threads (per row and element) that share the heads
  int* error_flag;
};

template <bool VEC>
__global__ void __launch_bounds__(256) k_paged_rope_append(const AppendArgs a) {
  pdl_trigger();
  pdl_wait();
  constexpr int W = VEC ? 4 : 1;
  const int half = a.D >> 1, lanes = half / W, heads = a.H + 2 * a.KVH;
  const int64_t total = (int64_t)a.rows * a.groups * lanes;
  for (int64_t id = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; id < total; id += (int64_t)gridDim.x * blockDim.x) {
    const int64_t rest = id / lanes;
    const int j = (int)(id - rest * lanes) * W;
    const int t = (int)(rest / a.groups), group = (int)(rest - (int64_t)t * a.groups);
    int pos = 0, slot = -1;
    const bool pos_ok = integral(a.pos[t * a.pos_s], 0, a.tab_rows - 1, pos);
    if (!integral(a.slot[t * a.slot_s], -1, a.slots - 1, slot)) {
      slot = -1;
      if (j == 0 && group == 0) atomicExch(a.error_flag, 73);
    }
    if (!pos_ok) {
      slot = -1;
      if (j == 0 && group == 0) atomicExch(a.error_flag, 72);
    }
    float c0[W], c1[W], s0[W], s1[W];
    auto get = [](const float* p, float* x) {
      if (VEC) {
        const float4 f = *reinterpret_cast<const float4*>(p);
        x[0] = f.x; x[1 % W] = f.y; x[2 % W] = f.z; x[3 % W] = f.w;
      } else {
        x[0] = *p;
      }
    };
    auto put = [](float* p, const float* x) {
      if (VEC) *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1 % W], x[2 % W], x[3 % W]);
      else *p = x[0];
    };
    if (pos_ok) {
      const float* cr = a.cos + (int64_t)pos * a.tab + j;
      const float* sr = a.sin + (int64_t)pos * a.tab + j;
      get(cr, c0);
      get(cr + half, c1);
      get(sr, s0);
      get(sr + half, s1);
    }
    const int page = slot >= 0 ? a.page.div(slot) : 0;
    const int64_t at = (int64_t)page * a.c0 + (int64_t)(slot - page * a.page.size) * a.c2 + j;
    for (int h = group; h < heads; h += a.groups) {
      const float* src;
      float* dst;
      const bool is_v = h >= a.H + a.KVH;
      if (h < a.H) {
        src = a.q + (int64_t)t * a.q0 + (int64_t)h * a.q1 + j;
        dst = a.q_out + ((int64_t)t * a.H + h) * a.D + j;
      } else if (slot < 0) {
        break;  // k and v of a row without a slot
      } else if (!is_v) {
        src = a.k + (int64_t)t * a.k0 + (int64_t)(h - a.H) * a.k1 + j;
        dst = a.kc + at + (int64_t)(h - a.H) * a.c1;
      } else {
        src = a.v + (int64_t)t * a.v0 + (int64_t)(h - a.H - a.KVH) * a.v1 + j;
        dst = a.vc + at + (int64_t)(h - a.H - a.KVH) * a.c1;
      }
      float x0[W], x1[W];
      if (!pos_ok) {
#pragma unroll
        for (int e = 0; e < W; e++) x0[e] = x1[e] = 0.0f;
      } else {
        get(src, x0);
        get(src + half, x1);
        if (!is_v) {
#pragma unroll
          for (int e = 0; e < W; e++) {
            const float y0 = __fadd_rn(__fmul_rn(x0[e], c0[e]), __fmul_rn(-x1[e], s0[e]));
            x1[e] = __fadd_rn(__fmul_rn(x1[e], c1[e]), __fmul_rn(x0[e], s1[e]));
            x0[e] = y0;
          }
        }
      }
      put(dst, x0);
      put(dst + half, x1);
    }
  }
}

}  // namespace paged
}  // namespace pai

using namespace pai;

PAI_API pai_status pai_paged_plan(pai_ctx* ctx, const pai_tensor* lengths, const pai_tensor* new_tokens,
                                  const pai_tensor* table, const pai_tensor* ring, const pai_tensor* state,
                                  int32_t page_size, int32_t rows, pai_tensor* q_start, pai_tensor* kv_len,
                                  pai_tensor* slots, pai_tensor* positions, pai_tensor* next_state) {
  PAI_TRY(enter(ctx));
  std::lock_guard<std::recursive_mutex> lk(ctx->mu);
  const pai_tensor* ins[5] = {lengths, new_tokens, table, ring, state};
  const char* names[5] = {"lengths", "new_tokens", "table", "ring", "state"};
  for (int i = 0; i < 5; i++) PAI_TRY(check_view(ctx, ins[i], names[i]));
  PAI_TRY(pai_paged::check_plan(set_error, lengths, new_tokens, table, ring, state, page_size, rows));
  const int n = lengths->dims[0];
  const int32_t d1 = n + 1, dn = n, dr = rows, d2 = 2;
  const int32_t* dims[5] = {&d1, &dn, &dr, &dr, &d2};
  Results<5> r(ctx);
  for (int i = 0; i < 5; i++) PAI_TRY(r.add(1, dims[i]));
  paged::PlanArgs a{};
  a.len = fptr(*lengths); a.len_s = lengths->strides[0];
  a.add = fptr(*new_tokens); a.add_s = new_tokens->strides[0];
  a.table = fptr(*table); a.t0 = table->strides[0]; a.t1 = table->strides[1];
  a.ring = fptr(*ring); a.ring_s = ring->strides[0];
  a.state = fptr(*state); a.state_s = state->strides[0];
  a.n = n; a.max_pages = table->dims[1]; a.pages = ring->dims[0]; a.rows = rows;
  a.per = (n + paged::kPlanThreads - 1) / paged::kPlanThreads;
  a.page = paged::page_div(page_size);
  a.q_start = fptr(r.t[0]); a.kv_len = fptr(r.t[1]); a.slots = fptr(r.t[2]); a.positions = fptr(r.t[3]); a.next_state = fptr(r.t[4]);
  a.error_flag = ctx->d_error_flag;
  PAI_PDL_LAUNCH(launch_pdl(paged::k_paged_plan, dim3(grid_for(ctx, rows, paged::kPlanThreads, 1, 2)),
                            dim3(paged::kPlanThreads), 0, ctx->stream, a),
                 "paged plan");
  *q_start = r.take(0); *kv_len = r.take(1); *slots = r.take(2); *positions = r.take(3); *next_state = r.take(4);
  return PAI_OK;
}

PAI_API pai_status pai_paged_rope_append(pai_ctx* ctx, const pai_tensor* q, const pai_tensor* k, const pai_tensor* v,
                                         const pai_tensor* cos_table, const pai_tensor* sin_table,
                                         const pai_tensor* positions, const pai_tensor* slots, const pai_tensor* k_cache,
                                         const pai_tensor* v_cache, pai_tensor* q_out) {
  PAI_TRY(enter(ctx));
  std::lock_guard<std::recursive_mutex> lk(ctx->mu);
  const pai_tensor* ins[9] = {q, k, v, cos_table, sin_table, positions, slots, k_cache, v_cache};
  const char* names[9] = {"q", "k", "v", "cos", "sin", "positions", "slots", "k_cache", "v_cache"};
  for (int i = 0; i < 9; i++) PAI_TRY(check_view(ctx, ins[i], names[i]));
  PAI_TRY(pai_paged::check_append(set_error, q, k, v, cos_table, sin_table, positions, slots, k_cache, v_cache));
  Results<1> r(ctx);
  PAI_TRY(r.add(3, q->dims));
  paged::AppendArgs a{};
  a.q = fptr(*q); a.q0 = q->strides[0]; a.q1 = q->strides[1];
  a.k = fptr(*k); a.k0 = k->strides[0]; a.k1 = k->strides[1];
  a.v = fptr(*v); a.v0 = v->strides[0]; a.v1 = v->strides[1];
  a.cos = fptr(*cos_table); a.sin = fptr(*sin_table); a.tab = cos_table->strides[0];
  a.pos = fptr(*positions); a.pos_s = positions->strides[0];
  a.slot = fptr(*slots); a.slot_s = slots->strides[0];
  a.kc = fptr(*k_cache); a.vc = fptr(*v_cache);
  a.c0 = k_cache->strides[0]; a.c1 = k_cache->strides[1]; a.c2 = k_cache->strides[2];
  a.q_out = fptr(r.t[0]);
  a.rows = q->dims[0]; a.H = q->dims[1]; a.KVH = k->dims[1]; a.D = q->dims[2];
  a.tab_rows = cos_table->dims[0]; a.slots = k_cache->dims[0] * k_cache->dims[2];
  a.page = paged::page_div(k_cache->dims[2]);
  a.error_flag = ctx->d_error_flag;
  const int heads = a.H + 2 * a.KVH;
  if (a.rows > 0) {
    const bool vec = a.D % 8 == 0 && paged::aligned(*q) && paged::aligned(*k) && paged::aligned(*v) &&
                     paged::aligned(*cos_table) && paged::aligned(*sin_table) && paged::aligned(*k_cache) &&
                     paged::aligned(*v_cache);
    const int lanes = a.D / 2 / (vec ? 4 : 1);
    // One head per thread until the grid fills the GPU, then up to 8, which share one read of the tables, position and
    // slot: 32 rows of 48 heads of 64, 4.2 us with one head (replayed graph), 4.3 with four, 6.3 with eight; 13,657 rows 77, 62
    // and 63 us.
    const int64_t threads = (int64_t)a.rows * heads * lanes;
    int64_t share = threads / ((int64_t)ctx->sm_count * 2048);
    share = share < 1 ? 1 : share > 8 ? 8 : share;
    a.groups = (int)((heads + share - 1) / share);
    const int64_t total = (int64_t)a.rows * a.groups * lanes;
    const dim3 grid(grid_for(ctx, total, 256, 1, 64));
    PAI_PDL_LAUNCH(vec ? launch_pdl(paged::k_paged_rope_append<true>, grid, dim3(256), 0, ctx->stream, a)
                       : launch_pdl(paged::k_paged_rope_append<false>, grid, dim3(256), 0, ctx->stream, a),
                   "paged rope append");
  }
  *q_out = r.take(0);
  return PAI_OK;
}
