// Causal attention of a step's new tokens over a paged KV cache (entry point pai_sdpa_paged): requests of different
// lengths, each with its own chunk of new tokens, keys and values read through page tables.
//
//   o_t = sum_{j <= p_t} exp(s_tj - m_t) v_j / sum_{j <= p_t} exp(s_tj - m_t),  s_tj = scale q_t . k_j
//
// k_paged_rows serves few query rows per kv head: decode steps and small chunks. It computes in fp32 and reads each key and
// value once for all the rows of a kv head's group, about two multiply-adds per byte at four rows, so HBM bounds it: 32
// requests of 2,800 keys, 32 query heads over 8 kv heads of 64 (375 MB), 72 us = 5.2 TB/s, four of 39,000 (639 MB) 121 us.
// About 6 us of either are its start (reading the requests, listing the share, the first keys: a chain of reads) and its
// end; in between it reads 5.7 to 6 TB/s. Many rows take the tensor-core kernel of attention_paged_tc.cu.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "attention_paged.cuh"
#include "tc_common.cuh"

namespace pai {
namespace paged {

using tc::ex2_sfu;
using tc::smem_u32;

constexpr int kRowsThreads = 256;
constexpr int kRowsWarps = kRowsThreads / 32;
constexpr int kRowsPerSm = 2;  // resident blocks (registers)
constexpr int kUnit = 64;      // keys per unit of the work split
constexpr int kGroupKeys = 2;  // consecutive keys per lane group
constexpr float kRise = 8.0f;  // a row's reference follows its maximum when that is 2^kRise above it

__device__ __forceinline__ void copy_async16(void* to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void copy_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int PENDING>
__device__ __forceinline__ void copy_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory");
}

constexpr int kRingBytes = 12288;  // per warp

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
// LPK lanes hold one key's or value's head dims (NV float4 each) and the query rows' same dims in registers; a warp has
// 32 / LPK such groups with KH consecutive keys each. The KH * R partial dot products of a group are summed over its
// lanes by Scatter, which leaves each lane one (row, key) score to exponentiate; the probabilities go back to the
// group's lanes by shuffles for P V. Keys and values come through a ring in shared memory, which each lane fills by
// asynchronous copies two steps ahead (five with one float4 per lane) with what it reads itself, so the ring needs no barrier
// and the keys on their way (128 KB per SM, 160) no registers. Weights are taken against 2^8 above a reference that follows the row maximum only when
// that rises by 2^8, so the sums are hardly ever rescaled, and no weight is above 1: a large value, weighted, does not
// overflow. Steps of keys that every row attends have no masks, and where pages hold whole groups a group's page is looked
// up once.
//
// Work split: every (request, kv head, group of R rows) is ceil(len / 64) units; the units of all of them, in order,
// are divided evenly over the blocks, so lengths need not be alike. A block's share is a run of segments, listed in
// shared memory before the first begins: under load a dependent read takes 3,000 cycles and more, so the copies run on
// into the next segment while one ends, and its queries are read while the one before is computed. A segment that is a
// whole (request, kv head, rows) writes its result, a partial one goes to the block's slot in `part`, and the last of
// its blocks to arrive joins the slots in block order (the same sum whichever comes last).
struct Seg {
  int req, first, row0, rows, kvh, shift;  // request and its first row; rows of the group; p_t = shift + t
  int j0, jend, open;                      // keys j0 .. jend - 1; before `open`, every row attends every key
  int whole, c0, c1;                       // not split; first and last block of a split one
};
constexpr int kSegs = 32;  // listed at a time

template <int R, int LPK, int NV>
__global__ void __launch_bounds__(kRowsThreads, kRowsPerSm) k_paged_rows(const AttnArgs a) {
  constexpr int KH = kGroupKeys;
  constexpr int kGroups = 32 / LPK;       // key groups per warp
  constexpr int kStep = kGroups * KH;     // keys per warp step
  constexpr int kStride = kRowsWarps * kStep;
  constexpr int V = R * KH;
  using S = Scatter<V, LPK>;
  constexpr int kKeep = S::kKeep, kRep = S::kRep;
  constexpr int kOwn = kKeep >= KH ? kKeep / KH : 1;             // rows whose scores a lane keeps
  constexpr int kRowLanes = kKeep >= KH ? 1 : KH / kKeep;        // lanes (kRep apart) that share a row
  constexpr int kWidth = 4 * LPK * NV;                           // padded head dim
  constexpr int kOut = R * kWidth;
  constexpr int kSlot = kOut + 2 * R;
  constexpr int kStage = 2 * KH * NV * 32;                       // float4s of a warp's ring per step
  constexpr int kStages = kRingBytes / (16 * kStage);
  static_assert(kStages >= 3 && kStages * 4 <= 32, "copies ahead, and their bits in `wrong`");
  constexpr int kRound = kOut < kRowsThreads ? R : kRowsThreads / kWidth;  // rows whose parts are joined at a time
  constexpr int kQ = (kOut + kRowsThreads - 1) / kRowsThreads;
  extern __shared__ float4 s_ring[];  // [warp][stage][K, V][KH][NV][lane]
  __shared__ __align__(16) float s_acc[kRowsWarps][kRound][kWidth];
  __shared__ __align__(16) float s_q[R][kWidth];
  __shared__ float s_m[kRowsWarps][R], s_l[kRowsWarps][R];
  __shared__ int64_t s_tmp[2 * kRowsWarps];
  __shared__ int64_t s_pair[2];
  __shared__ Seg s_seg[kSegs], s_split[2];
  __shared__ int s_last[2], s_unplaced;  // a row range is invalid
  pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int grp = lane / LPK, gl = lane % LPK;
  const int d0 = 4 * gl;  // the lane's head dims: d0 + 4 LPK h ..+ 3

  auto units_of = [&](const Req& r, int& groups, int& tiles) -> int64_t {
    groups = r.n > 0 ? (int)(((int64_t)r.n * a.g + R - 1) / R) : 0;
    tiles = max(1, (r.len + kUnit - 1) / kUnit);
    return (int64_t)a.KVH * groups * tiles;
  };
  // the block's share of the units
  const int per = (a.n + kRowsThreads - 1) / kRowsThreads;
  const int i0 = min(a.n, tid * per), i1 = min(a.n, i0 + per);
  int64_t count[2] = {0, 0}, count_before[2], all[2];  // units, pairs (kv head, rows)
  int groups, tiles;
  Req r;
  bool placed = true;
  if (tid == 0) s_unplaced = 0;  // set behind block_prefix's barriers
  for (int i = i0; i < i1; i++) {
    if (!load_req(a, i, r)) atomicExch(a.error_flag, 74);
    placed = placed && r.placed;
    count[0] += units_of(r, groups, tiles);
    count[1] += (int64_t)a.KVH * groups;
  }
  block_prefix<kRowsThreads>(count, s_tmp, count_before, all);
  if (!placed) s_unplaced = 1;
  const int64_t total = all[0], before = count_before[0], pairs_before = count_before[1];
  const int64_t G = min((int64_t)gridDim.x, total), c = blockIdx.x;
  if (c >= G) {
    __syncthreads();
    if (!s_unplaced) zero_rest(a);
    return;
  }
  const int64_t u0 = div_pos(c * total, G), u1 = div_pos((c + 1) * total, G);
  // the requests of this thread that have units in the block's share: f(request, its first unit, its first pair, its units)
  auto each = [&](auto f) {
    int64_t ub = before, pb = pairs_before;
    for (int i = i0; i < i1 && ub < u1; i++) {
      if (per > 1) load_req(a, i, r);
      const int64_t u = units_of(r, groups, tiles);
      if (u > 0 && ub + u > u0) f(i, ub, pb, u);
      ub += u;
      pb += (int64_t)a.KVH * groups;
    }
  };
  each([&](int, int64_t ub, int64_t pb, int64_t u) {
    if (ub <= u0) s_pair[0] = pb + div_pos(u0 - ub, tiles);
    if (u1 <= ub + u) s_pair[1] = pb + div_pos(u1 - 1 - ub, tiles);
  });

  auto store = [&](const Seg& g, int y, int d, float A, float L) {
    if (y < g.rows && d < a.D) {
      const int s = a.heads.div(g.row0 + y), h = g.kvh * a.g + (g.row0 + y) - s * a.g;
      a.out[((int64_t)(g.first + s) * a.H + h) * a.D + d] = L == 0.0f ? 0.0f : A / L;
    }
  };
  float4* const ring = s_ring + warp * (kStages * kStage) + lane;
  if (d0 + 4 * LPK * (NV - 1) >= a.D) {  // nothing is copied for lanes past the head dims
#pragma unroll 1
    for (int x = 0; x < kStages * 2 * KH * NV; x++) ring[x * 32] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  __syncthreads();
  const int64_t p0 = s_pair[0];
  const int segs = (int)(s_pair[1] - p0) + 1;
  bool bad_page = false;
  int splits = 0;

  for (int base = 0; base < segs; base += kSegs) {
    const int ns = min(kSegs, segs - base);
    each([&](int i, int64_t ub, int64_t pb, int64_t u) {
      const int64_t lo = max(u0, ub) - ub, hi = min(u1, ub + u) - ub;
      const int64_t first = max(pb + div_pos(lo, tiles), p0 + base), last = min(pb + div_pos(hi - 1, tiles), p0 + base + ns - 1);
      for (int64_t pair = first; pair <= last; pair++) {
        Seg g;
        const int64_t at = ub + (pair - pb) * tiles;  // the pair's first unit
        const int tile0 = (int)(max(u0, at) - at), tile1 = (int)(min(u1, at + tiles) - at);
        g.req = i;
        g.first = r.first;
        g.kvh = (int)(pair - pb) / groups;
        g.row0 = ((int)(pair - pb) - g.kvh * groups) * R;
        g.rows = (int)min((int64_t)R, (int64_t)r.n * a.g - g.row0);
        g.shift = r.len - r.n;
        g.j0 = tile0 * kUnit;
        g.jend = min(tile1 * kUnit, g.shift + a.heads.div(g.row0 + g.rows - 1) + 1);
        g.open = min(g.jend, g.shift + a.heads.div(g.row0) + 1);
        g.whole = tile0 == 0 && tile1 == tiles;
        g.c0 = g.c1 = (int)c;
        if (at < u0) g.c0 = (int)div_pos((at + 1) * G - 1, total);
        if (at + tiles > u1) g.c1 = (int)div_pos((at + tiles) * G - 1, total);
        s_seg[pair - p0 - base] = g;
      }
    });
    __syncthreads();

    // the queries of a segment, scaled so that scores are powers of two
    float qn[kQ];
    auto read_q = [&](const Seg& g) {
#pragma unroll
      for (int i = 0; i < kQ; i++) {
        const int t = tid + i * kRowsThreads, y = t / kWidth, d = t % kWidth;
        qn[i] = 0.0f;
        if (t < kOut && y < g.rows && d < a.D) {
          const int s = a.heads.div(g.row0 + y), head = g.kvh * a.g + (g.row0 + y) - s * a.g;
          qn[i] = a.q[(int64_t)(g.first + s) * a.q0 + (int64_t)head * a.q1 + d];
        }
      }
    };
    auto write_q = [&] {
#pragma unroll
      for (int i = 0; i < kQ; i++) {
        const int t = tid + i * kRowsThreads;
        if (t < kOut) s_q[t / kWidth][t % kWidth] = fmaf(qn[i], a.scale_hi, qn[i] * a.scale_lo);
      }
    };

    // what the copies read next: step ld_j (a warp's groups' keys are KH apart) of segment ld
    int ld = -1, ld_j = 0, ld_end = 0;
    const float* trow = nullptr;
    int64_t head_off = 0;
    float id = 0.0f;      // of the page of the lane's first key there
    unsigned wrong = 0;   // four bits per stage: the keys whose page is named wrongly
    auto advance = [&] {
      ld_j += kStride;
      while (ld_j >= ld_end && ++ld < ns) {
        const Seg& g = s_seg[ld];
        ld_j = g.j0 + warp * kStep;
        ld_end = g.jend;
        trow = a.table + (int64_t)g.req * a.t0;
        head_off = (int64_t)g.kvh * a.c1 + d0;
      }
      if (ld < ns) id = trow[a.page.div(min(ld_j + grp * KH, ld_end - 1)) * a.t1];
    };
    // Starts the copies of the lane's part of that step's KH keys and values into stage `st`. Keys that do not exist or
    // whose page is named wrongly are zero or unused.
    auto stage = [&](int st) {
      wrong &= ~(15u << (4 * st));
      if (ld < ns) {
        const int jg = ld_j + grp * KH;
        float4* to = ring + st * kStage;
        if (a.whole_groups && ld_j + kStep <= ld_end) {
          int page;
          if (!integral(id, 0, a.pages - 1, page)) {
            wrong |= 15u << (4 * st);
            page = 0;
          }
          const int64_t at = (int64_t)page * a.c0 + (jg - a.page.div(jg) * a.page.size) * a.c2 + head_off;
          const float* kp = a.k + at;
          const float* vp = a.v + at;
#pragma unroll
          for (int h = 0; h < NV; h++)
            if (d0 + 4 * LPK * h < a.D) {
#pragma unroll
              for (int e = 0; e < KH; e++) {
                copy_async16(to + (e * NV + h) * 32, kp + e * a.c2 + 4 * LPK * h);
                copy_async16(to + ((KH + e) * NV + h) * 32, vp + e * a.c2 + 4 * LPK * h);
              }
            }
        } else {
#pragma unroll 1
          for (int e = 0; e < KH; e++) {
            int64_t at = -1;
            if (jg + e < ld_end) {
              const int pi = a.page.div(jg + e);
              int page;
              if (integral(trow[pi * a.t1], 0, a.pages - 1, page))
                at = (int64_t)page * a.c0 + (int64_t)(jg + e - pi * a.page.size) * a.c2 + head_off;
              else
                wrong |= 1u << (4 * st + e);
            }
#pragma unroll 1
            for (int h = 0; h < NV; h++) {
              const int d = d0 + 4 * LPK * h;
              const float* kp = a.k + at + 4 * LPK * h;
              const float* vp = a.v + at + 4 * LPK * h;
              float4 kf = make_float4(0.f, 0.f, 0.f, 0.f), vf = kf;
              if (at >= 0 && a.vec) {
                if (d < a.D) {
                  kf = *reinterpret_cast<const float4*>(kp);
                  vf = *reinterpret_cast<const float4*>(vp);
                }
              } else if (at >= 0) {
                if (d < a.D) { kf.x = kp[0]; vf.x = vp[0]; }
                if (d + 1 < a.D) { kf.y = kp[1]; vf.y = vp[1]; }
                if (d + 2 < a.D) { kf.z = kp[2]; vf.z = vp[2]; }
                if (d + 3 < a.D) { kf.w = kp[3]; vf.w = vp[3]; }
              }
              to[(e * NV + h) * 32] = kf;
              to[((KH + e) * NV + h) * 32] = vf;
            }
          }
        }
        bad_page = bad_page || wrong != 0;
        advance();
      }
      copy_async_commit();
    };

    read_q(s_seg[0]);
    advance();
#pragma unroll
    for (int x = 0; x < kStages - 1; x++) stage(x);
    write_q();
    __syncthreads();
    int turn = 0;
    for (int x = 0; x < ns; x++) {
      const Seg& g = s_seg[x];
      float4 qv[R][NV];
      float2 acc[R][2 * NV];
#pragma unroll
      for (int y = 0; y < R; y++)
#pragma unroll
        for (int h = 0; h < NV; h++) {
          qv[y][h] = *reinterpret_cast<const float4*>(&s_q[y][d0 + 4 * LPK * h]);
          acc[y][2 * h] = acc[y][2 * h + 1] = make_float2(0.f, 0.f);
        }
      if (x + 1 < ns) read_q(s_seg[x + 1]);
      float m[kOwn], ref[kOwn], l[kOwn];  // reference; kRise above it, or 0 while there is none; sum
      int limit[kOwn];                    // the last key that each kept score's row attends
#pragma unroll
      for (int o = 0; o < kOwn; o++) {
        const int y = S::base(gl) / KH + o;
        limit[o] = y < g.rows ? g.shift + a.heads.div(g.row0 + y) : -1;
        m[o] = -INFINITY;
        ref[o] = l[o] = 0.0f;
      }
      const int jend = g.jend, open = g.open;

      // Scores, weights and sums of a group's keys from jg on; MASKED: some row attends not all of them.
      auto compute = [&](auto masked, int jg, const float4* from, unsigned wrong_keys) {
        constexpr bool MASKED = decltype(masked)::value;
        float x[V];
#pragma unroll
        for (int e = 0; e < KH; e++) {
          float4 kf[NV];
#pragma unroll
          for (int h = 0; h < NV; h++) kf[h] = from[(e * NV + h) * 32];
#pragma unroll
          for (int y = 0; y < R; y++) {
            float2 t = __fmul2_rn(make_float2(qv[y][0].x, qv[y][0].y), make_float2(kf[0].x, kf[0].y));
            t = __ffma2_rn(make_float2(qv[y][0].z, qv[y][0].w), make_float2(kf[0].z, kf[0].w), t);
#pragma unroll
            for (int h = 1; h < NV; h++) {
              t = __ffma2_rn(make_float2(qv[y][h].x, qv[y][h].y), make_float2(kf[h].x, kf[h].y), t);
              t = __ffma2_rn(make_float2(qv[y][h].z, qv[y][h].w), make_float2(kf[h].z, kf[h].w), t);
            }
            x[y * KH + e] = t.x + t.y;
          }
        }
        S::run(x, gl);
        bool hidden = false, rise = false;
        if (MASKED) {
#pragma unroll
          for (int i = 0; i < kKeep; i++) {
            const int e = (S::base(gl) + i) % KH;
            if (jg + e > limit[i / KH < kOwn ? i / KH : 0] || ((wrong_keys >> e) & 1u)) {
              x[i] = -INFINITY;
              hidden = true;
            }
          }
        }
#pragma unroll
        for (int i = 0; i < kKeep; i++) rise = rise || x[i] > m[i / KH < kOwn ? i / KH : 0] + kRise;  // never on NaN
        if (__any_sync(0xffffffffu, rise)) {
          float alpha[kOwn];
#pragma unroll
          for (int o = 0; o < kOwn; o++) {
            float mx = m[o];
#pragma unroll
            for (int i = 0; i < kKeep; i++)
              if (kOwn == 1 || i / KH == o) mx = fmaxf(mx, x[i]);
#pragma unroll
            for (int sh = kRep; sh < kRep * kRowLanes; sh <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, sh));
            if (mx > m[o] + kRise) {
              alpha[o] = ex2_sfu(m[o] - mx);
              m[o] = mx;
              ref[o] = mx + kRise;
              l[o] *= alpha[o];
            } else {
              alpha[o] = 1.0f;
            }
          }
#pragma unroll
          for (int y = 0; y < R; y++) {
            const float f = __shfl_sync(0xffffffffu, alpha[(y * KH % kKeep) / KH < kOwn ? (y * KH % kKeep) / KH : 0],
                                        S::lane_of(y * KH), LPK);
#pragma unroll
            for (int h = 0; h < 2 * NV; h++) acc[y][h] = __fmul2_rn(acc[y][h], make_float2(f, f));
          }
        }
        float p[kKeep];
#pragma unroll
        for (int i = 0; i < kKeep; i++) {
          const int o = i / KH < kOwn ? i / KH : 0;
          p[i] = ex2_sfu(x[i] - ref[o]);  // a NaN score stays one
          l[o] += p[i];
        }
        // a hidden key's value may be NaN or infinite: it is skipped, not multiplied by 0
        const bool any_hidden = MASKED && __any_sync(0xffffffffu, hidden);
#pragma unroll
        for (int e = 0; e < KH; e++) {
          float4 vf[NV];
#pragma unroll
          for (int h = 0; h < NV; h++) vf[h] = from[((KH + e) * NV + h) * 32];
#pragma unroll
          for (int y = 0; y < R; y++) {
            const int vi = y * KH + e;
            const float w = __shfl_sync(0xffffffffu, p[vi % kKeep], S::lane_of(vi), LPK);
            if (!any_hidden || w != 0.0f) {
#pragma unroll
              for (int h = 0; h < NV; h++) {
                acc[y][2 * h] = __ffma2_rn(make_float2(w, w), make_float2(vf[h].x, vf[h].y), acc[y][2 * h]);
                acc[y][2 * h + 1] = __ffma2_rn(make_float2(w, w), make_float2(vf[h].z, vf[h].w), acc[y][2 * h + 1]);
              }
            }
          }
        }
      };

      for (int j = g.j0 + warp * kStep; j < jend; j += kStride) {
        copy_async_wait<kStages - 2>();
        const unsigned wrong_keys = (wrong >> (4 * turn)) & 15u;
        stage(turn == 0 ? kStages - 1 : turn - 1);  // the step before has been read
        const float4* from = ring + turn * kStage;
        if (j + kStep <= open && __all_sync(0xffffffffu, wrong_keys == 0)) compute(std::false_type{}, j + grp * KH, from, 0u);
        else compute(std::true_type{}, j + grp * KH, from, wrong_keys);
        turn = turn + 1 == kStages ? 0 : turn + 1;
      }

      // join the warp's groups
#pragma unroll
      for (int o = 0; o < kOwn; o++)
#pragma unroll
        for (int sh = kRep; sh < kRep * kRowLanes; sh <<= 1) l[o] += __shfl_xor_sync(0xffffffffu, l[o], sh);
#pragma unroll
      for (int y = 0; y < R; y++) {
        constexpr int kLast = kOwn - 1;
        const int o = y * KH % kKeep / KH < kLast ? y * KH % kKeep / KH : kLast;
        const float my = __shfl_sync(0xffffffffu, m[o], S::lane_of(y * KH), LPK);
        float ly = __shfl_sync(0xffffffffu, l[o], S::lane_of(y * KH), LPK), M = my;
#pragma unroll
        for (int sh = LPK; sh < 32; sh <<= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, sh));
        const float f = M == -INFINITY ? 1.0f : ex2_sfu(my - M);
        ly *= f;
#pragma unroll
        for (int h = 0; h < 2 * NV; h++) acc[y][h] = __fmul2_rn(acc[y][h], make_float2(f, f));
#pragma unroll
        for (int sh = LPK; sh < 32; sh <<= 1) {
          ly += __shfl_xor_sync(0xffffffffu, ly, sh);
#pragma unroll
          for (int h = 0; h < 2 * NV; h++) {
            acc[y][h].x += __shfl_xor_sync(0xffffffffu, acc[y][h].x, sh);
            acc[y][h].y += __shfl_xor_sync(0xffffffffu, acc[y][h].y, sh);
          }
        }
        if (lane == 0) {
          s_m[warp][y] = M;
          s_l[warp][y] = ly;
        }
      }
      // ... and the warps
      float* slot = a.part + (size_t)(2 * c + (c == g.c0 ? 1 : 0)) * kSlot;
#pragma unroll
      for (int y0 = 0; y0 < R; y0 += kRound) {
        if (grp == 0) {
#pragma unroll
          for (int y = 0; y < kRound; y++)
#pragma unroll
            for (int h = 0; h < NV; h++)
              *reinterpret_cast<float4*>(&s_acc[warp][y][d0 + 4 * LPK * h]) = make_float4(
                  acc[y0 + y][2 * h].x, acc[y0 + y][2 * h].y, acc[y0 + y][2 * h + 1].x, acc[y0 + y][2 * h + 1].y);
        }
        __syncthreads();
        if (y0 == 0 && x + 1 < ns) write_q();  // this segment's are in registers
        if (tid < kRound * kWidth) {
          const int y = y0 + tid / kWidth, d = tid % kWidth;
          float M = -INFINITY, A = 0.0f, L = 0.0f;
#pragma unroll
          for (int w = 0; w < kRowsWarps; w++) M = fmaxf(M, s_m[w][y]);
#pragma unroll
          for (int w = 0; w < kRowsWarps; w++) {
            const float f = M == -INFINITY ? 1.0f : ex2_sfu(s_m[w][y] - M);
            L += s_l[w][y] * f;
            A += s_acc[w][y - y0][d] * f;
          }
          if (g.whole) {
            store(g, y, d, A, L);
          } else {
            slot[y * kWidth + d] = A;
            if (d == 0) { slot[kOut + y] = M; slot[kOut + R + y] = L; }
          }
        }
        __syncthreads();
      }
      if (!g.whole) {  // the block's first segment, its last or both
        if (tid == 0) s_split[splits] = g;
        splits++;
      }
    }
    copy_async_wait<0>();
    __syncthreads();  // the list has been read
  }

  if (!s_unplaced) zero_rest(a);
  if (splits > 0) {
    __threadfence();
    __syncthreads();
    if (tid < splits) {
      const Seg& g = s_split[tid];
      s_last[tid] = atomicAdd(&a.tickets[g.c0], 1u) == (unsigned)(g.c1 - g.c0);
      if (s_last[tid]) a.tickets[g.c0] = 0;
    }
    __syncthreads();
    for (int k = 0; k < splits; k++) {
      if (!s_last[k]) continue;
      const Seg& g = s_split[k];
      __threadfence();
      for (int t = tid; t < kOut; t += kRowsThreads) {
        const int y = t / kWidth, d = t % kWidth;
        float M = -INFINITY, A = 0.0f, L = 0.0f;
#pragma unroll 8
        for (int b = g.c0; b <= g.c1; b++)
          M = fmaxf(M, __ldcg(a.part + (size_t)(2 * b + (b == g.c0 ? 1 : 0)) * kSlot + kOut + y));
#pragma unroll 8
        for (int b = g.c0; b <= g.c1; b++) {
          const float* sl = a.part + (size_t)(2 * b + (b == g.c0 ? 1 : 0)) * kSlot;
          const float f = M == -INFINITY ? 1.0f : ex2_sfu(__ldcg(sl + kOut + y) - M);
          L += __ldcg(sl + kOut + R + y) * f;
          A += __ldcg(sl + t) * f;
        }
        store(g, y, d, A, L);
      }
    }
  }
  if (bad_page) atomicExch(a.error_flag, 75);
}

template <int R, int LPK, int NV>
static cudaError_t launch_rows(pai_ctx* ctx, const AttnArgs& a, int grid) {
  constexpr int bytes = kRowsWarps * kRingBytes;
  cudaError_t e = smem_limit(ctx, k_paged_rows<R, LPK, NV>, bytes);
  return e != cudaSuccess ? e : launch_pdl(k_paged_rows<R, LPK, NV>, dim3(grid), dim3(kRowsThreads), bytes, ctx->stream, a);
}

// Up to four rows a lane holds eight head dims, which halves the shuffles per key; the registers of eight rows leave no
// room for that.
template <int R>
static cudaError_t launch_rows(pai_ctx* ctx, const AttnArgs& a, int grid) {
  if (a.D <= 16) return launch_rows<R, 4, 1>(ctx, a, grid);
  if constexpr (R <= 4) {
    if (a.D <= 32) return launch_rows<R, 4, 2>(ctx, a, grid);
    if (a.D <= 64) return launch_rows<R, 8, 2>(ctx, a, grid);
    return launch_rows<R, 16, 2>(ctx, a, grid);
  } else {
    if (a.D <= 32) return launch_rows<R, 8, 1>(ctx, a, grid);
    if (a.D <= 64) return launch_rows<R, 16, 1>(ctx, a, grid);
    return launch_rows<R, 32, 1>(ctx, a, grid);
  }
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
  Results<1> r(ctx);
  PAI_TRY(r.add(3, q->dims));
  paged::AttnArgs a{};
  a.q = fptr(*q); a.q0 = q->strides[0]; a.q1 = q->strides[1];
  a.k = fptr(*k_cache); a.v = fptr(*v_cache);
  a.c0 = k_cache->strides[0]; a.c1 = k_cache->strides[1]; a.c2 = k_cache->strides[2];
  a.table = fptr(*table); a.t0 = table->strides[0]; a.t1 = table->strides[1];
  a.start = fptr(*q_start); a.start_s = q_start->strides[0];
  a.len = fptr(*kv_len); a.len_s = kv_len->strides[0];
  a.out = fptr(r.t[0]);
  a.n = table->dims[0]; a.rows = q->dims[0]; a.H = q->dims[1]; a.D = q->dims[2];
  a.KVH = k_cache->dims[1]; a.g = a.H / a.KVH; a.heads = paged::page_div(a.g);
  a.pages = k_cache->dims[0]; a.max_pages = table->dims[1];
  a.max_new = max_new > 0 ? std::min(max_new, a.rows) : a.rows;
  a.page = paged::page_div(k_cache->dims[2]);
  const double scale2 = (double)scale * 1.4426950408889634;
  a.scale_hi = (float)scale2;
  a.scale_lo = (float)(scale2 - (double)a.scale_hi);
  a.tickets = ctx->d_tickets;
  a.error_flag = ctx->d_error_flag;
  if (numel(r.t[0]) > 0) {
    a.vec = a.D % 4 == 0 && paged::aligned(*k_cache) && paged::aligned(*v_cache);
    a.q_vec = a.D % 4 == 0 && paged::aligned(*q);
    a.whole_groups = a.vec && a.page.size % paged::kGroupKeys == 0 && a.pages > 0;
    // Rows of one kv head: up to 8 the fp32 kernel reads each key once for all of them. Above, it would read keys again
    // for every 8 rows and its multiply-adds bound it; the tensor-core kernel's time hardly depends on the rows up to 128.
    // Measured by replayed graphs, 16 requests of about 1,900 keys, 8 kv heads of 64, us (fp32, tensor cores): 4 rows 37, 56;
    // 8 rows 49, 56; 12 rows 75, 56; 24 rows 103, 57; 32 rows 133, 58; 12 kv heads, 8 rows 64, 74; 16 rows 104, 76.
    const int64_t most = (int64_t)a.max_new * a.g;
    const bool tc = most > 8 && paged::tc_fits(a);
    const int R = most <= 1 ? 1 : most <= 2 ? 2 : most <= 4 ? 4 : 8;
    // no more blocks than units there can be (a bound on them may pass 64 bits, not a double's range)
    const int64_t groups = (most + R - 1) / R, tiles = std::max<int64_t>(1, ((int64_t)a.max_pages * a.page.size + 63) / 64);
    const double units = std::max(1.0, (double)a.n * a.KVH) * (double)groups * (double)tiles;
    const int grid = (int)std::min((double)std::min(ctx->sm_count * paged::kRowsPerSm, kTickets), units);
    const int width = a.D <= 16 ? 16 : a.D <= 32 ? 32 : a.D <= 64 ? 64 : 128;
    Scratch part;
    PAI_TRY(scratch(ctx, tc ? paged::tc_part_bytes(ctx) : (size_t)grid * 2 * R * (width + 2) * 4, &part));
    a.part = static_cast<float*>(part.p);
    KernelTimerScope timer(ctx, "attn_paged", 0.0);
    if (tc) {
      PAI_TRY(paged::tc_launch(ctx, a));
    } else {
      cudaError_t e = R == 1   ? paged::launch_rows<1>(ctx, a, grid)
                      : R == 2 ? paged::launch_rows<2>(ctx, a, grid)
                      : R == 4 ? paged::launch_rows<4>(ctx, a, grid)
                               : paged::launch_rows<8>(ctx, a, grid);
      PAI_PDL_LAUNCH(e, "paged attention");
    }
  }
  *out = r.take(0);
  return PAI_OK;
}
