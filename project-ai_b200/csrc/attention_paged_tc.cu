// Paged attention on the tensor cores: requests with more query rows per kv head than the fp32 kernel
// (attention_paged.cu) is good for, i.e. chunks of new tokens.
//
// Arithmetic. A product of fp32 numbers is taken as three fp16 products: with x = hi + lo, hi = fp16(x) and
// lo = fp16(x - hi), x·y = hi·hi' + hi·lo' + lo·hi' up to 3·2^-22 relative, accumulated in fp32 by the tensor cores.
// fp16 holds 2^-24 .. 65504, so operands are first scaled by powers of two (exact) that bring the largest magnitude of
// a query row, or of a tile of 128 keys or values, to [2^13, 2^14); numbers far below that lose relative precision
// only under 2^-39 of the largest. The scales come out again in a factor that the softmax and the sum over tiles
// multiply by anyway. Weights are scaled by 2^14 for the same reason, in numerator and denominator alike. This is half
// the tensor time of three TF32 products and half the shared memory. Per tile of keys the product P·V goes to its own
// accumulator and is added to fp32 registers with the running rescale, so the tensor cores' sums stay short (24 steps).
//
// One persistent CTA per SM works on an item: 256 query rows (two tiles of 128, row = token * g + head of the group) of
// one (request, kv head) against a run of key tiles:
//   warps 0-3, 4-7  one softmax warpgroup per query tile, a thread per row: writes Q (split) to TMEM; per key tile takes
//                   the row maximum of S, exponentiates, writes P (split) over S in TMEM, and adds the last P·V to its
//                   64 registers of output while the tensor cores compute the next S;
//   warps 8-11      split K and V: read a raw fp32 tile from shared memory, write hi and lo (SWIZZLE_128B rows of 64)
//                   over it;
//   warp 12         copies raw K and V rows from their pages with bulk copies, up to three tiles ahead;
//   warps 13, 14    one thread each issues S = Q·Kᵀ and P·V of one query tile; while one tile is in its softmax the
//                   other's products run.
// Both query tiles use each converted K and V tile, which halves conversion and shared-memory writes per product.
//
// Work split: as in k_paged_rows, the (item, key tile) units of all requests in one line, divided evenly over the CTAs;
// an item that crosses CTAs leaves fp32 partial results that the last of them to finish joins in CTA order.
// Every wait is bounded; a timeout sets the context's error flag and the CTA drains and exits.
#include <cuda_fp16.h>

#include "attention_paged.cuh"
#include "tc_common.cuh"

namespace pai {
namespace paged {

using tc::bulk_g2s;
using tc::commit;
using tc::desc_sw128;
using tc::ex2_sfu;
using tc::fence_after;
using tc::fence_before;
using tc::mbar_arrive;
using tc::mbar_expect_tx;
using tc::mbar_init;
using tc::smem_u32;
using tc::tmem_ld32;
using tc::tmem_st32;
using tc::tmem_st_wait;

constexpr int kTcRows = 128;                 // query rows of one tile
constexpr int kTcKeys = 128;                 // keys of one tile
constexpr int kTcDim = 64;                   // padded head dim
constexpr int kTcStages = 3;                 // K and V tiles in shared memory
constexpr int kTcRing = 8;                   // scales of the last tiles (more than the tiles in flight between two readers)
constexpr int kTcThreads = 512;              // four warpgroups; the last warp is idle
constexpr int kConvWarp = 8, kLoadWarp = 12, kIssueWarp = 13;
// Registers per thread of the softmax, conversion and loading/issuing warpgroups: 2·168 + 104 + 64 = 504 of the
// 4·128 = 512 that the CTA is launched with.
constexpr int kSoftmaxRegs = 168, kConvRegs = 104, kMiscRegs = 64;
static_assert(2 * kSoftmaxRegs + kConvRegs + kMiscRegs <= 4 * 128, "more registers than the launch holds");
constexpr uint32_t kHalfTile = kTcKeys * 128;      // hi or lo: 128 rows of 64 fp16
constexpr uint32_t kTile = 2 * kHalfTile;          // 32 KB, the size of the raw fp32 tile as well
constexpr int kTcPart = 2 * kTcRows * (kTcDim + 2);  // floats of one partial result
// TMEM columns: S and P of both query tiles, their P·V, their Q (hi, lo: 32 columns each)
__host__ __device__ constexpr uint32_t col_s(int t) { return 128u * (uint32_t)t; }
__host__ __device__ constexpr uint32_t col_pv(int t) { return 256u + 64u * (uint32_t)t; }
__host__ __device__ constexpr uint32_t col_q(int t) { return 384u + 64u * (uint32_t)t; }

struct TcShared {
  uint64_t raw[2][kTcStages];    // [K, V]: the raw tile has landed
  uint64_t conv[2][kTcStages];   // it is split
  uint64_t empty[2][kTcStages];  // both query tiles' products have read it
  uint64_t s_full[2], p_full[2], pv_full[2], q_full[2], done[2], drained[2];  // per query tile
  int64_t tmp[kTcThreads / 32];
  int64_t off, total;
  uint32_t seen[kTcRing][4];     // keys of a tile that exist (bit per key)
  uint32_t max_bits[2][4];       // converter warps' largest magnitudes
  uint32_t odd[2][4];            // ... and whether a value is not finite
  float scale[2][kTcRing];       // what a product with the tile is multiplied by to undo the tile's scale
  int v_odd[kTcRing];            // a V tile held values that are not finite
  int req;
  volatile int abort;
  int last[2];
  uint32_t tmem;
};
constexpr int kTcSmem = 1024 + 2 * kTcStages * (int)kTile + (int)sizeof(TcShared);

// kind::f16 descriptors: fp16 operands, fp32 accumulator; b_mn: B stored with its N index contiguous.
__host__ __device__ constexpr uint32_t idesc_f16(int m, int n, bool b_mn) {
  return (1u << 4) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// D (TMEM) (+)= A (TMEM, two fp16 per column) · B (shared)
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc));
}

// Bounded wait that also gives up once another role of the CTA has.
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, const volatile int* abort) {
  const uint32_t addr = smem_u32(bar);
  for (uint32_t i = 0; i < tc::kWaitLimit; i++) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(addr), "r"(parity)
        : "memory");
    if (done) return true;
    if ((i & 255u) == 255u && *abort) return false;
  }
  return false;
}
// Lane 0 polls, the warp follows its result.
__device__ __forceinline__ bool warp_wait_bar(uint64_t* bar, uint32_t parity, const volatile int* abort) {
  int ok = 0;
  if ((threadIdx.x & 31) == 0) ok = wait_bar(bar, parity, abort) ? 1 : 0;
  return __shfl_sync(0xffffffffu, ok, 0) != 0;
}
__device__ __forceinline__ void bar_named(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// The power of two that brings a magnitude (bits of a finite fp32, sign cleared) to [2^13, 2^14), and its inverse.
// Magnitudes under 2^-112 keep the largest scale.
__device__ __forceinline__ void tile_scale(uint32_t bits, float& up, float& down) {
  const int e = bits == 0 ? 140 : max(14, (int)(bits >> 23));  // biased exponent
  up = __uint_as_float((uint32_t)(267 - e) << 23);
  down = __uint_as_float((uint32_t)(e - 13) << 23);
}
__device__ __forceinline__ bool finite_bits(uint32_t bits) { return bits < 0x7f800000u; }

__device__ __forceinline__ uint32_t pack2(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
// Two fp32 numbers as fp16 hi parts and fp16 remainders (first number in the low half).
__device__ __forceinline__ void split2(float x0, float x1, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(x0, x1);
  const float2 f = __half22float2(h);
  hi = pack2(h);
  lo = pack2(__floats2half2_rn(x0 - f.x, x1 - f.y));
}

// A request's units: per kv head, groups of 256 rows, each with the key tiles that its last row attends.
struct Shape {
  int rows, groups;  // per kv head
  int64_t units;     // of one kv head
};
__device__ __forceinline__ int group_tiles(const AttnArgs& a, const Req& r, int rows, int group) {
  const int last = min(rows, (group + 1) * 2 * kTcRows) - 1;
  const int keys = r.len - r.n + last / a.g + 1;  // that the group's last row attends
  return max(1, (keys + kTcKeys - 1) / kTcKeys);
}
__device__ __forceinline__ Shape shape_of(const AttnArgs& a, const Req& r) {
  Shape s;
  s.rows = r.n * a.g;
  s.groups = (s.rows + 2 * kTcRows - 1) / (2 * kTcRows);
  s.units = 0;
  for (int i = 0; i < s.groups; i++) s.units += group_tiles(a, r, s.rows, i);
  return s;
}

// One run of key tiles [t0, t1) of a row group; `tiles` are all of the group's.
struct Item {
  Req r;
  int req, kvh, row0, rows, t0, t1, tiles;
  int64_t unit;  // of tile 0, in the line of all units
};

// Walks the CTA's share of the units; every role walks it alike.
struct Walk {
  int req;
  int64_t off, u, u1;
  __device__ __forceinline__ bool next(const AttnArgs& a, Item& it) {
    while (u < u1) {
      load_req(a, req, it.r);
      const Shape s = shape_of(a, it.r);
      if (off >= s.units * a.KVH) {
        req++;
        off = 0;
        continue;
      }
      it.kvh = (int)(off / s.units);
      int64_t rest = off - it.kvh * s.units;
      int group = 0;
      for (;; group++) {
        it.tiles = group_tiles(a, it.r, s.rows, group);
        if (rest < it.tiles) break;
        rest -= it.tiles;
      }
      it.req = req;
      it.row0 = group * 2 * kTcRows;
      it.rows = s.rows;
      it.t0 = (int)rest;
      it.t1 = (int)min((int64_t)it.tiles, rest + (u1 - u));
      it.unit = u - rest;
      u += it.t1 - it.t0;
      off += it.t1 - it.t0;
      return true;
    }
    return false;
  }
};

// Key tiles of the item that query tile t (its first row `row0`) attends: [t0, result).
__device__ __forceinline__ int tile_end(const AttnArgs& a, const Item& it, int row0) {
  const int last = min(it.rows, row0 + kTcRows) - 1;
  const int keys = it.r.len - it.r.n + last / a.g + 1;
  return max(it.t0, min(it.t1, (keys + kTcKeys - 1) / kTcKeys));
}

// ---------------------------------------------------------------- roles
// Softmax warpgroup of query tile `tile`.
template <int tile>
__device__ __forceinline__ void softmax_role(const AttnArgs& a, TcShared& sh, Walk walk, uint32_t tmem) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = warp & 3;
  const int row = quad * 32 + lane;
  const uint32_t base = tmem + ((uint32_t)(quad * 32) << 16);
  const uint32_t cs = base + col_s(tile), cpv = base + col_pv(tile), cq = base + col_q(tile);
  const int64_t G = min((int64_t)gridDim.x, sh.total);
  bool ok = true;
  int J = 0, C = 0;  // key tiles of the CTA and of this query tile so far
  Item it;
  while (walk.next(a, it)) {
    const int first = it.row0 + tile * kTcRows;
    if (first >= it.rows) {
      J += it.t1 - it.t0;
      continue;
    }
    const int r = first + row;
    const bool live = r < it.rows;
    const int s = r / a.g, h = it.kvh * a.g + (r - s * a.g);
    const int limit = live ? it.r.len - it.r.n + s : -1;  // the last key this row attends
    const int first_limit = it.r.len - it.r.n + first / a.g;
    const int end = tile_end(a, it, first);
    float qdown;  // undoes the row's scale
    {
      float x[64];
      uint32_t big = 0;
      const float* p = a.q + (int64_t)(it.r.first + s) * a.q0 + (int64_t)h * a.q1;
      if (a.q_vec) {
#pragma unroll
        for (int d = 0; d < 64; d += 4) {
          const float4 v = live && d < a.D ? *reinterpret_cast<const float4*>(p + d) : make_float4(0.f, 0.f, 0.f, 0.f);
          x[d] = v.x; x[d + 1] = v.y; x[d + 2] = v.z; x[d + 3] = v.w;
        }
      } else {
#pragma unroll
        for (int d = 0; d < 64; d++) x[d] = live && d < a.D ? p[d] : 0.0f;
      }
#pragma unroll
      for (int d = 0; d < 64; d++) {
        x[d] = (float)((double)x[d] * a.scale2);  // scores in powers of two; rounded once from 64 bits
        const uint32_t b = __float_as_uint(x[d]) & 0x7fffffffu;
        if (finite_bits(b)) big = max(big, b);
      }
      float up;
      tile_scale(big, up, qdown);
      float lo[32];
#pragma unroll
      for (int d = 0; d < 32; d++) {
        uint32_t hi, l;
        split2(x[2 * d] * up, x[2 * d + 1] * up, hi, l);
        x[d] = __uint_as_float(hi);
        lo[d] = __uint_as_float(l);
      }
      if (ok) {
        tmem_st32(cq, x);
        tmem_st32(cq + 32, lo);
        tmem_st_wait();
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.q_full[tile]);
      }
    }
    float o[64];
#pragma unroll
    for (int d = 0; d < 64; d++) o[d] = 0.0f;
    float m = -INFINITY, l = 0.0f, alpha = 1.0f;
    int odd = 0;
    auto fold = [&](int slot) {  // o = o * alpha + (P·V of the last tile)
      const float f = sh.scale[1][slot];
      odd |= sh.v_odd[slot];
#pragma unroll
      for (int c = 0; c < 2; c++) {
        float pv[32];
        tmem_ld32(cpv + 32 * c, pv);
#pragma unroll
        for (int d = 0; d < 32; d++) o[32 * c + d] = fmaf(pv[d], f, o[32 * c + d] * alpha);
      }
    };
    for (int t = it.t0; t < end; t++) {
      const int slot = (J + t - it.t0) % kTcRing;
      if (t > it.t0) {
        if (ok && !warp_wait_bar(&sh.pv_full[tile], (C - 1) & 1, &sh.abort)) ok = false;
        if (ok) {
          fence_after();
          fold((slot + kTcRing - 1) % kTcRing);
        }
      }
      if (ok && !warp_wait_bar(&sh.s_full[tile], C & 1, &sh.abort)) ok = false;
      if (!ok) break;
      fence_after();
      // kept finite and above 0: a score of 0 or -inf times it stays one
      const float c = fminf(fmaxf(qdown * sh.scale[0][slot], 1.1754944e-38f), 3.4028235e38f);
      const int k0 = t * kTcKeys;
      uint32_t vis[4];
      bool masked = k0 + kTcKeys - 1 > first_limit;
#pragma unroll
      for (int g = 0; g < 4; g++) {
        const int n = limit - (k0 + 32 * g) + 1;  // keys of the chunk up to the row's last
        const uint32_t upto = n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u;
        vis[g] = sh.seen[slot][g];
        masked = masked || vis[g] != 0xffffffffu;
        vis[g] &= upto;
      }
      float mx = -INFINITY;
#pragma unroll
      for (int g = 0; g < 4; g++) {
        float x[32];
        tmem_ld32(cs + 32 * g, x);
        if (masked) {
#pragma unroll
          for (int i = 0; i < 32; i++) mx = fmaxf(mx, (vis[g] >> i) & 1u ? x[i] : -INFINITY);
        } else {
#pragma unroll
          for (int i = 0; i < 32; i++) mx = fmaxf(mx, x[i]);
        }
      }
      const float mn = fmaxf(m, mx * c);
      alpha = mn == m ? 1.0f : ex2_sfu(m - mn);
      const float ref = (mn == -INFINITY ? 0.0f : mn) - 14.0f;
      m = mn;
      float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int g = 0; g < 4; g++) {
        float x[32], y[32];
        tmem_ld32(cs + 32 * g, x);
        if (masked) {
#pragma unroll
          for (int i = 0; i < 32; i++) x[i] = (vis[g] >> i) & 1u ? x[i] : -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < 16; i++) {
          const float p0 = ex2_sfu(fmaf(x[2 * i], c, -ref)), p1 = ex2_sfu(fmaf(x[2 * i + 1], c, -ref));
          part[(2 * i) & 3] += p0;
          part[(2 * i + 1) & 3] += p1;
          uint32_t hi, lo;
          split2(p0, p1, hi, lo);
          y[i] = __uint_as_float(hi);
          y[16 + i] = __uint_as_float(lo);
        }
        tmem_st32(cs + 32 * g, y);  // over the scores just read: keys 32g.. as 16 columns of hi, 16 of lo
      }
      l = l * alpha + ((part[0] + part[1]) + (part[2] + part[3]));
      tmem_st_wait();
      fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.p_full[tile]);
      C++;
    }
    if (end > it.t0) {
      if (ok && !warp_wait_bar(&sh.pv_full[tile], (C - 1) & 1, &sh.abort)) ok = false;
      if (ok) {
        fence_after();
        fold((J + end - 1 - it.t0) % kTcRing);
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.done[tile]);
      }
    }
    if (odd) {
      // Values that are not finite were left out of the products: add those that this row attends.
      const int k1 = min(it.t1 * kTcKeys, limit + 1);
      for (int j = it.t0 * kTcKeys; j < k1; j++) {
        const int pi = a.page.div(j);
        int page;
        if (!integral(a.table[it.req * a.t0 + pi * a.t1], 0, a.pages - 1, page)) continue;
        const float* v = a.v + (int64_t)page * a.c0 + (int64_t)it.kvh * a.c1 + (int64_t)(j - pi * a.page.size) * a.c2;
#pragma unroll
        for (int d = 0; d < 64; d++)
          if (d < a.D && !finite_bits(__float_as_uint(v[d]) & 0x7fffffffu)) o[d] += v[d];
      }
    }
    J += it.t1 - it.t0;
    const bool whole = it.t0 == 0 && it.t1 == it.tiles;
    float* out = a.out + ((int64_t)(it.r.first + s) * a.H + h) * a.D;
    auto store = [&](float sum) {
      const float inv = 1.0f / sum;
#pragma unroll
      for (int d = 0; d < 64; d += 4) {
        if (d < a.D) {
          const float4 v = make_float4(o[d] * inv, o[d + 1] * inv, o[d + 2] * inv, o[d + 3] * inv);
          *reinterpret_cast<float4*>(out + d) = sum == 0.0f ? make_float4(0.f, 0.f, 0.f, 0.f) : v;
        }
      }
    };
    if (whole) {
      if (ok && live) store(l);
      continue;
    }
    const int c0 = (int)(((it.unit + 1) * G - 1) / sh.total), c1 = (int)(((it.unit + it.tiles) * G - 1) / sh.total);
    auto slot_of = [&](int b) { return a.part + (size_t)(2 * b + (b == c0 ? 1 : 0)) * kTcPart; };
    float* mine = slot_of(blockIdx.x) + (size_t)(tile * kTcRows + row) * (kTcDim + 2);
#pragma unroll
    for (int d = 0; d < 64; d += 2) *reinterpret_cast<float2*>(mine + d) = make_float2(o[d], o[d + 1]);
    *reinterpret_cast<float2*>(mine + 64) = make_float2(m, l);
    __threadfence();
    bar_named(2 + tile, 128);
    if (row == 0) {
      unsigned* ticket = &a.tickets[2 * c0 + tile];
      sh.last[tile] = atomicAdd(ticket, 1u) == (unsigned)(c1 - c0);
      if (sh.last[tile]) *ticket = 0;
    }
    bar_named(2 + tile, 128);
    if (sh.last[tile]) {
      __threadfence();
      float M = -INFINITY, L = 0.0f;
      for (int b = c0; b <= c1; b++)
        M = fmaxf(M, __ldcg(slot_of(b) + (size_t)(tile * kTcRows + row) * (kTcDim + 2) + 64));
#pragma unroll
      for (int d = 0; d < 64; d++) o[d] = 0.0f;
      for (int b = c0; b <= c1; b++) {
        const float* p = slot_of(b) + (size_t)(tile * kTcRows + row) * (kTcDim + 2);
        const float2 ml = __ldcg(reinterpret_cast<const float2*>(p + 64));
        const float f = M == -INFINITY ? 1.0f : ex2_sfu(ml.x - M);
        L += ml.y * f;
#pragma unroll
        for (int d = 0; d < 64; d += 2) {
          const float2 v = __ldcg(reinterpret_cast<const float2*>(p + d));
          o[d] += v.x * f;
          o[d + 1] += v.y * f;
        }
      }
      if (ok && live) store(L);
    }
  }
  if (!ok && lane == 0) {
    atomicExch(a.error_flag, 76);
    sh.abort = 1;
  }
}

// Splits the raw K and V tiles in place.
__device__ __forceinline__ void convert_role(const AttnArgs& a, TcShared& sh, uint8_t* tiles, Walk walk) {
  const int tid = threadIdx.x - 32 * kConvWarp, warp = tid >> 5, lane = tid & 31;
  const int tr = tid >> 4, tc4 = tid & 15;  // 16 threads per row, 8 rows per pass
  bool ok = true;
  int J = 0;
  Item it;
  while (walk.next(a, it)) {
    for (int t = it.t0; t < it.t1; t++, J++) {
      const int st = J % kTcStages, slot = J % kTcRing;
      for (int op = 0; op < 2; op++) {
        uint8_t* tile = tiles + (op * kTcStages + st) * kTile;
        float4 x[16];
        uint32_t big = 0;
        bool odd = false;
        if (ok && !warp_wait_bar(&sh.raw[op][st], (J / kTcStages) & 1, &sh.abort)) ok = false;
        if (ok) {
          const float* raw = reinterpret_cast<const float*>(tile);
#pragma unroll
          for (int p = 0; p < 16; p++) {
            const int r = p * 8 + tr;
            const bool have = ((sh.seen[slot][p >> 2] >> (r & 31)) & 1u) && 4 * tc4 < a.D;
            x[p] = have ? *reinterpret_cast<const float4*>(raw + r * a.D + 4 * tc4) : make_float4(0.f, 0.f, 0.f, 0.f);
          }
#pragma unroll
          for (int p = 0; p < 16; p++) {
            const float v[4] = {x[p].x, x[p].y, x[p].z, x[p].w};
#pragma unroll
            for (int e = 0; e < 4; e++) {
              const uint32_t b = __float_as_uint(v[e]) & 0x7fffffffu;
              big = max(big, b);
            }
          }
          odd = !finite_bits(big);
          if (odd) {  // the largest finite magnitude
            big = 0;
#pragma unroll
            for (int p = 0; p < 16; p++) {
              const float v[4] = {x[p].x, x[p].y, x[p].z, x[p].w};
#pragma unroll
              for (int e = 0; e < 4; e++) {
                const uint32_t b = __float_as_uint(v[e]) & 0x7fffffffu;
                if (finite_bits(b)) big = max(big, b);
              }
            }
          }
        }
        big = __reduce_max_sync(0xffffffffu, big);
        odd = __any_sync(0xffffffffu, odd);
        if (lane == 0) {
          sh.max_bits[op][warp] = big;
          sh.odd[op][warp] = odd;
        }
        bar_named(1, 128);  // the maxima are there, and every thread holds its part of the raw tile
        if (!ok) continue;
        big = max(max(sh.max_bits[op][0], sh.max_bits[op][1]), max(sh.max_bits[op][2], sh.max_bits[op][3]));
        odd = (sh.odd[op][0] | sh.odd[op][1] | sh.odd[op][2] | sh.odd[op][3]) != 0;
        float up, down;
        tile_scale(big, up, down);
        if (tid == 0) {
          sh.scale[op][slot] = down;
          if (op == 1) sh.v_odd[slot] = odd;
        }
#pragma unroll
        for (int p = 0; p < 16; p++) {
          const int r = p * 8 + tr;
          float4 y = make_float4(x[p].x * up, x[p].y * up, x[p].z * up, x[p].w * up);
          if (odd && op == 1) {  // a value that is not finite would spoil the rows that do not attend it, too
            if (!isfinite(y.x)) y.x = 0.0f;
            if (!isfinite(y.y)) y.y = 0.0f;
            if (!isfinite(y.z)) y.z = 0.0f;
            if (!isfinite(y.w)) y.w = 0.0f;
          }
          uint2 hi, lo;
          split2(y.x, y.y, hi.x, lo.x);
          split2(y.z, y.w, hi.y, lo.y);
          uint8_t* dst = tile + r * 128 + (((tc4 >> 1) ^ (r & 7)) << 4) + ((tc4 & 1) << 3);
          *reinterpret_cast<uint2*>(dst) = hi;
          *reinterpret_cast<uint2*>(dst + kHalfTile) = lo;
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.conv[op][st]);
      }
    }
  }
  if (!ok && lane == 0) {
    atomicExch(a.error_flag, 77);
    sh.abort = 1;
  }
}

// Copies the raw K and V tiles out of their pages.
__device__ __forceinline__ void load_role(const AttnArgs& a, TcShared& sh, uint8_t* tiles, Walk walk) {
  const int lane = threadIdx.x & 31;
  const int P = a.page.size;
  const uint32_t row_bytes = (uint32_t)a.D * 4;
  bool ok = true, bad = false, copied_k = false;
  int J = 0;
  Item it;
  while (ok && walk.next(a, it)) {
    const float* trow = a.table + (int64_t)it.req * a.t0;
    const int64_t head = (int64_t)it.kvh * a.c1;
    for (int t = it.t0; t < it.t1; t++) {
      const int st = J % kTcStages, slot = J % kTcRing;
      const uint32_t parity = ((J / kTcStages) & 1) ^ 1;
      const int k0 = t * kTcKeys, k1 = min(k0 + kTcKeys, it.r.len);
      const int p0 = a.page.div(k0), p1 = k1 > k0 ? a.page.div(k1 - 1) : p0 - 1;
      uint32_t seen[4] = {0, 0, 0, 0};
      int count = 0;
      for (int pi = p0 + lane; pi <= p1; pi += 32) {
        int page;
        if (!integral(trow[pi * a.t1], 0, a.pages - 1, page)) {
          bad = true;
          continue;
        }
        const int lo = max(pi * P, k0) - k0, hi = min((pi + 1) * P, k1) - k0;  // key rows of the tile
        count += hi - lo;
#pragma unroll
        for (int g = 0; g < 4; g++) {
          const int x0 = max(lo - 32 * g, 0), x1 = min(hi - 32 * g, 32);
          if (x0 < x1) seen[g] |= (x1 - x0 == 32 ? 0xffffffffu : ((1u << (x1 - x0)) - 1u) << x0);
        }
      }
      count = __reduce_add_sync(0xffffffffu, count);
#pragma unroll
      for (int g = 0; g < 4; g++) seen[g] = __reduce_or_sync(0xffffffffu, seen[g]);
      for (int op = 0; op < 2 && ok; op++) {
        if (!warp_wait_bar(&sh.empty[op][st], parity, &sh.abort)) {
          ok = false;
          break;
        }
        uint8_t* tile = tiles + (op * kTcStages + st) * kTile;
        if (lane == 0) {
          if (op == 0) {
#pragma unroll
            for (int g = 0; g < 4; g++) sh.seen[slot][g] = seen[g];
          }
          mbar_expect_tx(&sh.raw[op][st], (uint32_t)count * row_bytes);
        }
        __syncwarp();
        copied_k = true;
        const float* src = (op == 0 ? a.k : a.v) + head;
        for (int pi = p0 + lane; pi <= p1; pi += 32) {
          int page;
          if (!integral(trow[pi * a.t1], 0, a.pages - 1, page)) continue;
          const int j0 = max(pi * P, k0), j1 = min((pi + 1) * P, k1);
          const float* from = src + (int64_t)page * a.c0 + (int64_t)(j0 - pi * P) * a.c2;
          uint8_t* to = tile + (uint32_t)(j0 - k0) * row_bytes;
          if (a.c2 == a.D) {
            bulk_g2s(to, from, (uint32_t)(j1 - j0) * row_bytes, &sh.raw[op][st]);
          } else {
            for (int j = j0; j < j1; j++) bulk_g2s(to + (uint32_t)(j - j0) * row_bytes, from + (int64_t)(j - j0) * a.c2, row_bytes, &sh.raw[op][st]);
          }
        }
      }
      if (!ok) break;
      J++;
      copied_k = false;
    }
  }
  if (bad) atomicExch(a.error_flag, 75);
  if (!ok && lane == 0) {
    atomicExch(a.error_flag, 78);
    sh.abort = 1;
  }
  // every product has signalled its stage, or at least every copy has landed, before the CTA may exit
  if (lane == 0) {
    for (int j = max(0, J - kTcStages); j <= J; j++) {
      for (int op = 0; op < 2; op++) {
        const int st = j % kTcStages;
        const uint32_t parity = (j / kTcStages) & 1;
        if (j == J) {  // a K tile copied without its V tile, when a wait gave up in between
          if (!ok && copied_k && op == 0) tc::mbar_wait(&sh.raw[0][st], parity);
        } else if (!wait_bar(&sh.empty[op][st], parity, &sh.abort)) {
          tc::mbar_wait(&sh.raw[op][st], parity);
        }
      }
    }
  }
}

// Issues the products of one query tile.
__device__ __forceinline__ void issue_role(const AttnArgs& a, TcShared& sh, uint8_t* tiles, Walk walk, uint32_t tmem, int tile) {
  constexpr uint32_t is = idesc_f16(kTcRows, kTcKeys, false), ip = idesc_f16(kTcRows, kTcDim, true);
  const uint32_t cs = tmem + col_s(tile), cpv = tmem + col_pv(tile), cq = tmem + col_q(tile);
  const uint32_t k_tiles = smem_u32(tiles), v_tiles = k_tiles + kTcStages * kTile;
  bool ok = true;
  int J = 0, C = 0, items = 0, dones = 0;
  Item it;
  auto skip = [&](int op, int j) {  // a tile this query tile does not use: free it once it is converted
    const int st = j % kTcStages;
    if (!wait_bar(&sh.conv[op][st], (j / kTcStages) & 1, &sh.abort)) return false;
    mbar_arrive(&sh.empty[op][st]);
    return true;
  };
  while (ok && walk.next(a, it)) {
    const int first = it.row0 + tile * kTcRows;
    const bool active = first < it.rows;
    const int end = active ? tile_end(a, it, first) : it.t0;
    if (active) {
      if (!wait_bar(&sh.q_full[tile], items & 1, &sh.abort)) { ok = false; break; }
      items++;
    }
    for (int t = it.t0; t < end; t++, J++) {
      const int st = J % kTcStages;
      const uint32_t parity = (J / kTcStages) & 1;
      if (!wait_bar(&sh.conv[0][st], parity, &sh.abort) ||
          (C > 0 && !wait_bar(&sh.pv_full[tile], (C - 1) & 1, &sh.abort))) {  // the last P has been read: S may replace it
        ok = false;
        break;
      }
      fence_after();
      const uint32_t kh = k_tiles + st * kTile, kl = kh + kHalfTile;
#pragma unroll
      for (int i = 0; i < 4; i++) mma_f16_ts(cs, cq + 32 + 8 * i, desc_sw128(kh + 32 * i), is, i > 0);
#pragma unroll
      for (int i = 0; i < 4; i++) mma_f16_ts(cs, cq + 8 * i, desc_sw128(kl + 32 * i), is, 1u);
#pragma unroll
      for (int i = 0; i < 4; i++) mma_f16_ts(cs, cq + 8 * i, desc_sw128(kh + 32 * i), is, 1u);
      commit(&sh.s_full[tile]);
      commit(&sh.empty[0][st]);
      if (!wait_bar(&sh.p_full[tile], C & 1, &sh.abort) || !wait_bar(&sh.conv[1][st], parity, &sh.abort)) {
        ok = false;
        break;
      }
      fence_after();
      const uint32_t vh = v_tiles + st * kTile, vl = vh + kHalfTile;
      // 16 keys per product: columns 32 (i / 2) + 8 (i % 2) of P's hi part, 16 further of its lo part
#pragma unroll
      for (int i = 0; i < 8; i++) mma_f16_ts(cpv, cs + 32 * (i >> 1) + 8 * (i & 1) + 16, desc_sw128(vh + 2048 * i), ip, i > 0);
#pragma unroll
      for (int i = 0; i < 8; i++) mma_f16_ts(cpv, cs + 32 * (i >> 1) + 8 * (i & 1), desc_sw128(vl + 2048 * i), ip, 1u);
#pragma unroll
      for (int i = 0; i < 8; i++) mma_f16_ts(cpv, cs + 32 * (i >> 1) + 8 * (i & 1), desc_sw128(vh + 2048 * i), ip, 1u);
      commit(&sh.pv_full[tile]);
      commit(&sh.empty[1][st]);
      C++;
    }
    // The softmax has read the last scales before this thread frees tiles that the ring's slots are reused for.
    if (ok && end > it.t0 && !wait_bar(&sh.done[tile], dones++ & 1, &sh.abort)) ok = false;
    for (int t = end; t < it.t1 && ok; t++, J++) ok = skip(0, J) && skip(1, J);
  }
  if (!ok) {
    atomicExch(a.error_flag, 79);
    sh.abort = 1;
  }
  // every product this thread issued completes before the CTA gives its tensor memory back
  commit(&sh.drained[tile]);
  tc::mbar_wait(&sh.drained[tile], 0);
}

__global__ void __launch_bounds__(kTcThreads, 1) k_paged_tc(const AttnArgs a) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* tiles = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  TcShared& sh = *reinterpret_cast<TcShared*>(tiles + 2 * kTcStages * kTile);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int op = 0; op < 2; op++)
      for (int i = 0; i < kTcStages; i++) {
        mbar_init(&sh.raw[op][i], 1);
        mbar_init(&sh.conv[op][i], 4);
        mbar_init(&sh.empty[op][i], 2);
      }
    for (int t = 0; t < 2; t++) {
      mbar_init(&sh.s_full[t], 1);
      mbar_init(&sh.p_full[t], 4);
      mbar_init(&sh.pv_full[t], 1);
      mbar_init(&sh.q_full[t], 4);
      mbar_init(&sh.done[t], 4);
      mbar_init(&sh.drained[t], 1);
    }
    sh.abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) tc::tmem_alloc(&sh.tmem, 512);
  pdl_trigger();
  pdl_wait();
  zero_rest(a);

  // this CTA's share of the units
  const int per = (a.n + kTcThreads - 1) / kTcThreads;
  const int i0 = min(a.n, tid * per), i1 = min(a.n, i0 + per);
  int64_t mine = 0, total;
  for (int i = i0; i < i1; i++) {
    Req r;
    if (!load_req(a, i, r)) atomicExch(a.error_flag, 74);
    mine += shape_of(a, r).units * a.KVH;
  }
  const int64_t before = block_prefix<kTcThreads>(mine, sh.tmp, total);
  const int64_t G = min((int64_t)gridDim.x, total), c = blockIdx.x;
  Walk walk{0, 0, 0, 0};
  if (c < G) {
    walk.u = c * total / G;
    walk.u1 = (c + 1) * total / G;
    if (before <= walk.u && walk.u < before + mine) {
      int64_t off = walk.u - before;
      for (int i = i0; i < i1; i++) {
        Req r;
        load_req(a, i, r);
        const int64_t units = shape_of(a, r).units * a.KVH;
        if (off < units) {
          sh.req = i;
          sh.off = off;
          sh.total = total;
          break;
        }
        off -= units;
      }
    }
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = sh.tmem;
  if (c < G) {
    walk.req = sh.req;
    walk.off = sh.off;
    if (warp < kConvWarp) {
      asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
      if (warp < 4) softmax_role<0>(a, sh, walk, tmem);
      else softmax_role<1>(a, sh, walk, tmem);
    } else if (warp < kLoadWarp) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kConvRegs));
      convert_role(a, sh, tiles, walk);
    } else {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kMiscRegs));
      if (warp == kLoadWarp) load_role(a, sh, tiles, walk);
      else if (warp < kIssueWarp + 2 && lane == 0) issue_role(a, sh, tiles, walk, tmem, warp - kIssueWarp);
    }
  }
  fence_before();
  __syncthreads();
  if (warp == 0) {
    fence_after();
    tc::tmem_dealloc(tmem, 512);
  }
}

// Aligned caches and a head dim of at most 64: bulk copies need 16-byte rows.
bool tc_fits(const AttnArgs& a) { return a.vec && a.D <= kTcDim && (int64_t)a.max_new * a.g < (1 << 30); }

size_t tc_part_bytes(const pai_ctx* ctx) { return (size_t)ctx->sm_count * 2 * kTcPart * 4; }

pai_status tc_launch(pai_ctx* ctx, const AttnArgs& a) {
  PAI_CUDA(smem_limit(ctx, k_paged_tc, kTcSmem));
  PAI_PDL_LAUNCH(launch_pdl(k_paged_tc, dim3(ctx->sm_count), dim3(kTcThreads), kTcSmem, ctx->stream, a),
                 "paged attention (tcgen05)");
  return PAI_OK;
}

}  // namespace paged
}  // namespace pai
