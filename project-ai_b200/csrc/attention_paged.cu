// Causal attention of a step's new tokens over a paged KV cache (entry point pai_sdpa_paged): requests of different
// lengths, each with its own chunk of new tokens, keys and values read through page tables.
//
//   o_t = sum_{j <= p_t} exp(s_tj - m_t) v_j / sum_{j <= p_t} exp(s_tj - m_t),  s_tj = scale q_t . k_j
//
// k_paged_rows (this file's first kernel) serves few query rows per kv head: decode steps and small chunks. It computes
// in fp32 and reads each key and value once for all the rows of a kv head's group, about two multiply-adds per byte at
// four rows, so HBM bounds it.
#include <math.h>

#include <algorithm>

#include "attention_paged.cuh"

namespace pai {
namespace paged {

constexpr int kRowsThreads = 256;
constexpr int kRowsWarps = kRowsThreads / 32;
constexpr int kRowsPerSm = 2;  // resident blocks (registers)
constexpr int kUnit = 64;      // keys per unit of the work split

// V values per lane, summed over the L lanes of a group: each lane is left with max(1, V / L) of the sums, value
// index base(lane) + i. Each step halves the values a lane keeps and sends the other half to its partner.
template <int V, int L>
struct Scatter {
  static constexpr int kKeep = V > L ? V / L : 1;
  static constexpr int kRep = V < L ? L / V : 1;  // lanes that end with the same value
  static __device__ __forceinline__ void run(float (&x)[V], int lane) {
    int cnt = V;
#pragma unroll
    for (int off = L / 2; off > 0; off >>= 1) {
      if (cnt > 1) {
        cnt /= 2;
        const bool up = (lane & off) != 0;
#pragma unroll
        for (int i = 0; i < V / 2; i++) {
          if (i < cnt) {
            const float send = up ? x[i] : x[i + cnt];
            const float keep = up ? x[i + cnt] : x[i];
            x[i] = keep + __shfl_xor_sync(0xffffffffu, send, off);
          }
        }
      } else {
        x[0] += __shfl_xor_sync(0xffffffffu, x[0], off);
      }
    }
  }
  static __device__ __forceinline__ int base(int lane) { return lane / kRep * kKeep; }      // lane within the group
  static __device__ __forceinline__ constexpr int lane_of(int v) { return v / kKeep * kRep; }
};

// R query rows of one kv head (token-major: row = token * g + head of the group) against its keys.
//
// LPK lanes hold one key's or value's head dims (a float4 each) and the query rows' same dims in registers; a warp has
// 32 / LPK such groups with KH consecutive keys each. The KH * R partial dot products of a group are summed over its
// lanes by Scatter, which leaves each lane one (row, key) score to exponentiate; the probabilities go back to the
// group's lanes by shuffles for P V. Nothing passes through shared memory until a segment ends, and the next keys'
// loads are in flight while these are computed.
//
// Work split: every (request, kv head, group of R rows) is ceil(len / 64) units; the units of all of them, in order,
// are divided evenly over the blocks, so lengths need not be alike. A block's share is a run of segments; a segment
// that is a whole (request, kv head, rows) writes its result, a partial one goes to the block's slot in `part`, and the
// last of its blocks to arrive joins the slots in block order (the same sum whichever comes last).
template <int R, int KH, int LPK>
__global__ void __launch_bounds__(kRowsThreads, kRowsPerSm) k_paged_rows(const AttnArgs a) {
  constexpr int kGroups = 32 / LPK;       // key groups per warp
  constexpr int kStep = kGroups * KH;     // keys per warp step
  constexpr int kStride = kRowsWarps * kStep;
  constexpr int V = R * KH;
  using S = Scatter<V, LPK>;
  constexpr int kKeep = S::kKeep, kRep = S::kRep;
  constexpr int kOwn = kKeep >= KH ? kKeep / KH : 1;             // rows whose scores a lane keeps
  constexpr int kRowLanes = kKeep >= KH ? 1 : KH / kKeep;        // lanes (kRep apart) that share a row
  constexpr int kWidth = 4 * LPK;                                // padded head dim
  constexpr int kParts = kRowsWarps * kGroups;
  constexpr int kSlot = R * (kWidth + 2);
  __shared__ float s_acc[kParts][R][kWidth];
  __shared__ float s_m[kParts][R], s_l[kParts][R];
  __shared__ int64_t s_tmp[kRowsWarps];
  __shared__ int64_t s_off;
  __shared__ int s_req, s_last;
  pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int grp = lane / LPK, gl = lane % LPK;
  const int d0 = 4 * gl;

  zero_rest(a);
  auto units_of = [&](const Req& r, int& groups, int& tiles) -> int64_t {
    groups = (int)(((int64_t)r.n * a.g + R - 1) / R);
    tiles = max(1, (r.len + kUnit - 1) / kUnit);
    return r.n > 0 ? (int64_t)a.KVH * groups * tiles : 0;
  };
  // the block's share of the units, and the request it starts in
  const int per = (a.n + kRowsThreads - 1) / kRowsThreads;
  const int i0 = min(a.n, tid * per), i1 = min(a.n, i0 + per);
  int64_t mine = 0, total;
  int groups, tiles;
  for (int i = i0; i < i1; i++) {
    Req r;
    if (!load_req(a, i, r)) atomicExch(a.error_flag, 74);
    mine += units_of(r, groups, tiles);
  }
  const int64_t before = block_prefix<kRowsThreads>(mine, s_tmp, total);
  const int64_t G = min((int64_t)gridDim.x, total), c = blockIdx.x;
  if (c >= G) return;
  const int64_t u0 = c * total / G, u1 = (c + 1) * total / G;
  if (before <= u0 && u0 < before + mine) {
    int64_t off = u0 - before;
    for (int i = i0; i < i1; i++) {
      Req r;
      load_req(a, i, r);
      const int64_t u = units_of(r, groups, tiles);
      if (off < u) { s_req = i; s_off = off; break; }
      off -= u;
    }
  }
  __syncthreads();
  int req = s_req;
  int64_t off = s_off;
  bool bad_page = false;

  for (int64_t u = u0; u < u1;) {
    Req r;
    load_req(a, req, r);
    const int64_t units = units_of(r, groups, tiles);
    if (off >= units) { req++; off = 0; continue; }
    const int64_t pair = off / tiles;
    const int tile0 = (int)(off - pair * tiles);
    const int tile1 = (int)min((int64_t)tiles, tile0 + (u1 - u));
    const int kvh = (int)(pair / groups), row0 = (int)(pair - (int64_t)kvh * groups) * R;
    const int nrows = (int)min((int64_t)R, (int64_t)r.n * a.g - row0);

    // query rows, scaled so that scores are powers of two
    float4 qv[R];
#pragma unroll
    for (int x = 0; x < R; x++) {
      qv[x] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (x < nrows) {
        const int s = (row0 + x) / a.g, h = kvh * a.g + (row0 + x) - s * a.g;
        const float* p = a.q + (int64_t)(r.first + s) * a.q0 + (int64_t)h * a.q1 + d0;
        if (d0 < a.D) qv[x].x = fmaf(p[0], a.scale_hi, p[0] * a.scale_lo);
        if (d0 + 1 < a.D) qv[x].y = fmaf(p[1], a.scale_hi, p[1] * a.scale_lo);
        if (d0 + 2 < a.D) qv[x].z = fmaf(p[2], a.scale_hi, p[2] * a.scale_lo);
        if (d0 + 3 < a.D) qv[x].w = fmaf(p[3], a.scale_hi, p[3] * a.scale_lo);
      }
    }
    // the last key that each kept score's row attends
    int limit[kOwn];
#pragma unroll
    for (int o = 0; o < kOwn; o++) {
      const int x = S::base(gl) / KH + o;
      limit[o] = x < nrows ? r.len - r.n + (row0 + x) / a.g : -1;
    }
    const int most = r.len - r.n + (row0 + nrows - 1) / a.g;  // the last row's
    const int jend = min(tile1 * kUnit, most + 1);

    float4 acc[R];
    float m[kOwn], l[kOwn];
#pragma unroll
    for (int x = 0; x < R; x++) acc[x] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int o = 0; o < kOwn; o++) { m[o] = -INFINITY; l[o] = 0.0f; }

    const float* trow = a.table + (int64_t)req * a.t0;
    const int64_t head_off = (int64_t)kvh * a.c1 + d0;
    // keys j .. j+KH-1 of this lane's group; bit e of `seen` is set where key j + e exists
    auto load = [&](int j, float4 (&kf)[KH], float4 (&vf)[KH]) -> unsigned {
      unsigned seen = 0;
#pragma unroll
      for (int e = 0; e < KH; e++) {
        kf[e] = vf[e] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (j + e < jend) {
          const int pi = a.page.div(j + e);
          int page;
          if (integral(trow[pi * a.t1], 0, a.pages - 1, page)) {
            seen |= 1u << e;
            const int64_t at = (int64_t)page * a.c0 + (int64_t)(j + e - pi * a.page.size) * a.c2 + head_off;
            if (a.vec) {
              if (d0 < a.D) {
                kf[e] = *reinterpret_cast<const float4*>(a.k + at);
                vf[e] = *reinterpret_cast<const float4*>(a.v + at);
              }
            } else {
              if (d0 < a.D) { kf[e].x = a.k[at]; vf[e].x = a.v[at]; }
              if (d0 + 1 < a.D) { kf[e].y = a.k[at + 1]; vf[e].y = a.v[at + 1]; }
              if (d0 + 2 < a.D) { kf[e].z = a.k[at + 2]; vf[e].z = a.v[at + 2]; }
              if (d0 + 3 < a.D) { kf[e].w = a.k[at + 3]; vf[e].w = a.v[at + 3]; }
            }
          } else {
            bad_page = true;
          }
        }
      }
      return seen;
    };

    float4 kf[KH], vf[KH];
    int j = tile0 * kUnit + warp * kStep;  // the warp's keys; its groups' are KH apart
    unsigned seen = load(j + grp * KH, kf, vf);
    while (j < jend) {
      float4 kn[KH], vn[KH];
      const unsigned seen_next = load(j + kStride + grp * KH, kn, vn);
      float x[V];
#pragma unroll
      for (int y = 0; y < R; y++)
#pragma unroll
        for (int e = 0; e < KH; e++)
          x[y * KH + e] = fmaf(qv[y].w, kf[e].w, fmaf(qv[y].z, kf[e].z, fmaf(qv[y].y, kf[e].y, qv[y].x * kf[e].x)));
      S::run(x, gl);
      const int jg = j + grp * KH;
      float p[kKeep];
      bool vis[kKeep], hidden = false, grew = false;
      float alpha[kOwn];
#pragma unroll
      for (int i = 0; i < kKeep; i++) {
        const int e = (S::base(gl) + i) % KH;
        vis[i] = ((seen >> e) & 1u) && jg + e <= limit[i / KH < kOwn ? i / KH : 0];
        hidden = hidden || !vis[i];
      }
#pragma unroll
      for (int o = 0; o < kOwn; o++) {
        float mx = m[o];
#pragma unroll
        for (int i = 0; i < kKeep; i++)
          if (kOwn == 1 || i / KH == o) mx = vis[i] ? fmaxf(mx, x[i]) : mx;
#pragma unroll
        for (int sh = kRep; sh < kRep * kRowLanes; sh <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, sh));
        alpha[o] = mx == m[o] ? 1.0f : pow2(m[o] - mx);
        grew = grew || mx != m[o];
        const float ref = mx == -INFINITY ? 0.0f : mx;  // no key so far: a NaN score stays one
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < kKeep; i++)
          if (kOwn == 1 || i / KH == o) {
            p[i] = vis[i] ? pow2(x[i] - ref) : 0.0f;
            sum += p[i];
          }
        l[o] = l[o] * alpha[o] + sum;
        m[o] = mx;
      }
      if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
        for (int y = 0; y < R; y++) {
          const float f = __shfl_sync(0xffffffffu, alpha[(y * KH % kKeep) / KH < kOwn ? (y * KH % kKeep) / KH : 0],
                                      S::lane_of(y * KH), LPK);
          acc[y].x *= f; acc[y].y *= f; acc[y].z *= f; acc[y].w *= f;
        }
      }
      // a hidden key's value may be NaN or infinite: it is skipped, not multiplied by 0
      const bool any_hidden = __any_sync(0xffffffffu, hidden);
#pragma unroll
      for (int y = 0; y < R; y++)
#pragma unroll
        for (int e = 0; e < KH; e++) {
          const int vi = y * KH + e;
          const float w = __shfl_sync(0xffffffffu, p[vi % kKeep], S::lane_of(vi), LPK);
          if (!any_hidden || w != 0.0f) {
            acc[y].x = fmaf(w, vf[e].x, acc[y].x);
            acc[y].y = fmaf(w, vf[e].y, acc[y].y);
            acc[y].z = fmaf(w, vf[e].z, acc[y].z);
            acc[y].w = fmaf(w, vf[e].w, acc[y].w);
          }
        }
#pragma unroll
      for (int e = 0; e < KH; e++) { kf[e] = kn[e]; vf[e] = vn[e]; }
      seen = seen_next;
      j += kStride;
    }

    // join the warps' groups
#pragma unroll
    for (int o = 0; o < kOwn; o++)
#pragma unroll
      for (int sh = kRep; sh < kRep * kRowLanes; sh <<= 1) l[o] += __shfl_xor_sync(0xffffffffu, l[o], sh);
    __syncthreads();  // the last segment's sums have been read
    const int part = warp * kGroups + grp;
#pragma unroll
    for (int y = 0; y < R; y++) {
      *reinterpret_cast<float4*>(&s_acc[part][y][d0]) = acc[y];
      if (gl == S::lane_of(y * KH)) {
        const int o = (y * KH % kKeep) / KH < kOwn ? (y * KH % kKeep) / KH : 0;
        s_m[part][y] = m[o];
        s_l[part][y] = l[o];
      }
    }
    __syncthreads();
    const bool whole = tile0 == 0 && tile1 == tiles;
    const int64_t first_unit = u - tile0, last_unit = first_unit + tiles - 1;  // of this pair, in the whole list
    const int c0 = (int)(((first_unit + 1) * G - 1) / total), c1 = (int)(((last_unit + 1) * G - 1) / total);
    auto store = [&](int y, int d, float A, float L) {
      if (y < nrows && d < a.D) {
        const int s = (row0 + y) / a.g, h = kvh * a.g + (row0 + y) - s * a.g;
        a.out[((int64_t)(r.first + s) * a.H + h) * a.D + d] = L == 0.0f ? 0.0f : A / L;
      }
    };
    float* slot = a.part + (size_t)(2 * c + (c == c0 ? 1 : 0)) * kSlot;
    for (int t = tid; t < R * kWidth; t += kRowsThreads) {
      const int y = t / kWidth, d = t % kWidth;
      float M = -INFINITY, A = 0.0f, L = 0.0f;
#pragma unroll
      for (int x = 0; x < kParts; x++) M = fmaxf(M, s_m[x][y]);
#pragma unroll
      for (int x = 0; x < kParts; x++) {
        const float f = M == -INFINITY ? 1.0f : pow2(s_m[x][y] - M);
        L += s_l[x][y] * f;
        A += s_acc[x][y][d] * f;
      }
      if (whole) {
        store(y, d, A, L);
      } else {
        slot[t] = A;
        if (d == 0) { slot[R * kWidth + y] = M; slot[R * kWidth + R + y] = L; }
      }
    }
    if (!whole) {
      __threadfence();
      __syncthreads();
      if (tid == 0) {
        s_last = atomicAdd(&a.tickets[c0], 1u) == (unsigned)(c1 - c0);
        if (s_last) a.tickets[c0] = 0;
      }
      __syncthreads();
      if (s_last) {
        __threadfence();
        for (int t = tid; t < R * kWidth; t += kRowsThreads) {
          const int y = t / kWidth, d = t % kWidth;
          float M = -INFINITY, A = 0.0f, L = 0.0f;
          for (int b = c0; b <= c1; b++)
            M = fmaxf(M, __ldcg(a.part + (size_t)(2 * b + (b == c0 ? 1 : 0)) * kSlot + R * kWidth + y));
#pragma unroll 4
          for (int b = c0; b <= c1; b++) {
            const float* sl = a.part + (size_t)(2 * b + (b == c0 ? 1 : 0)) * kSlot;
            const float f = M == -INFINITY ? 1.0f : pow2(__ldcg(sl + R * kWidth + y) - M);
            L += __ldcg(sl + R * kWidth + R + y) * f;
            A += __ldcg(sl + t) * f;
          }
          store(y, d, A, L);
        }
      }
    }
    u += tile1 - tile0;
    off += tile1 - tile0;
  }
  if (bad_page) atomicExch(a.error_flag, 75);
}

template <int LPK>
static cudaError_t launch_rows(const AttnArgs& a, int R, dim3 grid, cudaStream_t stream) {
  const dim3 block(kRowsThreads);
  if (R == 1) return launch_pdl(k_paged_rows<1, 4, LPK>, grid, block, 0, stream, a);
  if (R == 2) return launch_pdl(k_paged_rows<2, 4, LPK>, grid, block, 0, stream, a);
  if (R == 4) return launch_pdl(k_paged_rows<4, 4, LPK>, grid, block, 0, stream, a);
  return launch_pdl(k_paged_rows<8, 2, LPK>, grid, block, 0, stream, a);
}

}  // namespace paged
}  // namespace pai

using namespace pai;

PAI_API pai_status pai_sdpa_paged(pai_ctx* ctx, const pai_tensor* q, const pai_tensor* k_cache, const pai_tensor* v_cache,
                                  const pai_tensor* table, const pai_tensor* q_start, const pai_tensor* kv_len, float scale,
                                  int32_t max_new, pai_tensor* out) {
  PAI_TRY(enter(ctx));
  std::lock_guard<std::recursive_mutex> lk(ctx->mu);
  const pai_tensor* ins[6] = {q, k_cache, v_cache, table, q_start, kv_len};
  const char* names[6] = {"q", "k_cache", "v_cache", "table", "q_start", "kv_len"};
  for (int i = 0; i < 6; i++) PAI_TRY(check_view(ctx, ins[i], names[i]));
  PAI_TRY(pai_paged::check_sdpa(set_error, q, k_cache, v_cache, table, q_start, kv_len, max_new));
  pai_tensor r;
  PAI_TRY(alloc_tensor(ctx, 3, q->dims, PAI_F32, false, &r));
  paged::AttnArgs a{};
  a.q = fptr(*q); a.q0 = q->strides[0]; a.q1 = q->strides[1];
  a.k = fptr(*k_cache); a.v = fptr(*v_cache);
  a.c0 = k_cache->strides[0]; a.c1 = k_cache->strides[1]; a.c2 = k_cache->strides[2];
  a.table = fptr(*table); a.t0 = table->strides[0]; a.t1 = table->strides[1];
  a.start = fptr(*q_start); a.start_s = q_start->strides[0];
  a.len = fptr(*kv_len); a.len_s = kv_len->strides[0];
  a.out = fptr(r);
  a.n = table->dims[0]; a.rows = q->dims[0]; a.H = q->dims[1]; a.D = q->dims[2];
  a.KVH = k_cache->dims[1]; a.g = a.H / a.KVH;
  a.pages = k_cache->dims[0]; a.max_pages = table->dims[1];
  a.max_new = max_new > 0 ? std::min(max_new, a.rows) : a.rows;
  a.page = paged::page_div(k_cache->dims[2]);
  const double scale2 = (double)scale * 1.4426950408889634;
  a.scale_hi = (float)scale2;
  a.scale_lo = (float)(scale2 - (double)a.scale_hi);
  a.tickets = ctx->d_tickets;
  a.error_flag = ctx->d_error_flag;
  if (numel(r) > 0) {
    auto aligned = [](const pai_tensor& t) {
      if (reinterpret_cast<uintptr_t>(fptr(t)) % 16) return false;
      for (int i = 0; i + 1 < t.rank; i++)
        if (t.dims[i] > 1 && t.strides[i] % 4) return false;
      return true;
    };
    a.vec = a.D % 4 == 0 && aligned(*k_cache) && aligned(*v_cache);
    a.q_vec = a.D % 4 == 0 && aligned(*q);
    const int64_t most = (int64_t)a.max_new * a.g;  // rows of one kv head
    const bool tc = most > 8 && paged::tc_fits(a);
    const int R = most <= 1 ? 1 : most <= 2 ? 2 : most <= 4 ? 4 : 8;
    // no more blocks than units there can be
    const int64_t groups = (most + R - 1) / R, tiles = std::max<int64_t>(1, ((int64_t)a.max_pages * a.page.size + 63) / 64);
    const int64_t units = std::max<int64_t>(1, (int64_t)a.n * a.KVH) * groups * tiles;
    const int grid = (int)std::min<int64_t>(std::min(ctx->sm_count * paged::kRowsPerSm, kTickets), units);
    const int lanes = a.D <= 16 ? 4 : a.D <= 32 ? 8 : a.D <= 64 ? 16 : 32;
    Scratch part;
    PAI_TRY(scratch(ctx, tc ? paged::tc_part_bytes(ctx) : (size_t)grid * 2 * R * (4 * lanes + 2) * 4, &part));
    a.part = static_cast<float*>(part.p);
    KernelTimerScope timer(ctx, "attn_paged", 0.0);
    if (tc) {
      PAI_TRY(paged::tc_launch(ctx, a));
    } else {
      cudaError_t e = lanes == 4    ? paged::launch_rows<4>(a, R, dim3(grid), ctx->stream)
                      : lanes == 8  ? paged::launch_rows<8>(a, R, dim3(grid), ctx->stream)
                      : lanes == 16 ? paged::launch_rows<16>(a, R, dim3(grid), ctx->stream)
                                    : paged::launch_rows<32>(a, R, dim3(grid), ctx->stream);
      PAI_PDL_LAUNCH(e, "paged attention");
    }
  }
  *out = r;
  return PAI_OK;
}
