// Paged attention on the tensor cores: requests with more query rows per kv head than the fp32 kernel
// (attention_paged.cu) is good for, i.e. chunks of new tokens.
//
// Arithmetic. A product of fp32 numbers is taken as three fp16 products: with x = hi + lo, hi = fp16(x) and
// lo = fp16(x - hi), x·y = hi·hi' + hi·lo' + lo·hi' up to 3·2^-22 relative, accumulated in fp32 by the tensor cores. This
// is half the tensor time of three TF32 products and half the shared memory, but fp16 holds only 2^-24 .. 65504. So
//   q, K, V  are scaled by powers of two (exact) that bring the largest magnitude of a query row, or of a tile of 128 keys
//            or values, to [2^13, 2^14). A number is then off by 2^-22 of itself or 2^-39 of the largest, whichever is
//            more: the same for what lies within 2^16 of it. What a row does not attend shares the tile with what it does, so
//            a single large number, anywhere in it, would take the precision of all others. A tile of which some pair of
//            numbers (of a group of four adjacent ones) is more than 2^16 below the largest is therefore sorted: it takes the
//            scale that suits most keys (V, one for each head dim), and keys that do not fit are left out and added in fp32,
//            straight from their pages. Numbers thus count as in fp32 next to the largest of their group of four, which is
//            what the choice of keys goes by: single numbers of ordinary data are 2^16 below others often enough.
//            A row of q of which half of the groups or more are far below the largest makes keys fp32 work for its warp (all,
//            or those of uneven tiles); so do scores that could pass some thousand, where rounding is a matter of whole
//            powers of two, in tiles with values left out.
//   weights  exp(s - t) are taken against t, the power of two above the row's largest score in the tile, and times 2^14:
//            all they lose is 2^-38 of the tile's largest. (With t following the row's maximum only now and then, a tile of
//            small weights and large values lost all of them.) The factor from there to the row's reference, which does follow
//            only when the maximum has risen by 2^9, is an exact power of two and goes into the sums over tiles with the scale
//            of V. There weights are at most 1, so that a sum of large values does not overflow before it is divided.
// Per tile of keys the product P·V goes to its own accumulator and is added to fp32 registers, so the tensor cores' sums
// stay short (24 steps). Four chunks of 2,000 tokens over 2,000 cached ones, 0.66 ms, take 1.8 to 2.2 ms where all tiles are
// sorted (head dims of K or V that are always small), 1.1 with a large value in each of four pages, 4.4 with one in an eighth
// of the pages of 16, 8.6 in all; 107 if everything is fp32 work (one head dim of q or K 2^17 above all others).
//
// One persistent CTA per SM works on an item: 256 query rows (two tiles of 128, row = token * g + head of the group) of
// one (request, kv head) against a run of key tiles:
//   warps 0-7, 8-15 softmax of one query tile each, two threads per row (each half of the keys and half of the head
//                   dims): write Q (split) to TMEM; per key tile take the row maximum of S, exponentiate, write P (split)
//                   over S in TMEM, and add the last P·V to their 32 registers of output while the tensor cores compute
//                   the next S. The two groups take turns at this. (One thread per row left each scheduler one warp at
//                   this work, 336 cycles per 16 keys, most of it latency; two take 160 each, what the pipes need.)
//   warps 16-19, 20-23  split K and V: read a raw fp32 tile from shared memory, write hi and lo (SWIZZLE_128B rows of
//                   64) over it, eight rows at a time;
//   warp 24         copies raw K rows from their pages with bulk copies, up to three tiles ahead;
//   warps 25, 26    issue S = Q·Kᵀ and P·V of one query tile each;
//   warp 27         walks the CTA's share of the work, hands the items to the others, and copies V as warp 24 does K.
// Both query tiles use each converted K and V tile, which halves conversion and shared-memory writes per product. Up to
// 128 rows there is one query tile: both softmax groups then work on it, each on every second key tile; the second hands
// its result to the first through TMEM (six new tokens of 16 requests: 60 us, with one group 71; chunks among decoding
// requests 129 and 148).
//
// Measured, 32 query heads over 8 kv heads of 64 (times in this file are those of a replayed graph of the call): four chunks
// of 2,000 tokens over 2,000 cached ones 0.66 ms, 240 TFLOP/s of results (158 GFLOP), i.e. 720 of fp16 products. A key tile
// takes 8,400 cycles there: the chain of a query tile (scores 770 of tensor work, softmax 4,100, P·V 1,000, the waits
// between) with the other query tile's in the gaps, and half of the issue slots.
//
// Work split: as in k_paged_rows, the (item, key tile) units of all requests in one line, divided evenly over the CTAs;
// an item that crosses CTAs leaves fp32 partial results that the last of them to finish joins in CTA order.
// Every wait is bounded; a timeout sets the context's error flag and the CTA drains and exits.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "attention_paged.cuh"
#include "tc_common.cuh"

namespace pai {
namespace paged {

using tc::bulk_g2s;
using tc::commit;
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
constexpr int kSoftmaxWarps = 8;             // per query tile
constexpr int kConvWarps = 4;                // for K, and for V
constexpr int kConvWarp = 2 * kSoftmaxWarps, kLoadWarp = kConvWarp + 2 * kConvWarps, kIssueWarp = kLoadWarp + 1;
constexpr int kWalkWarp = kIssueWarp + 2;
constexpr int kTcThreads = 32 * (kWalkWarp + 1);  // seven warpgroups
constexpr int kItems = 4;                         // items handed out ahead
constexpr float kRise = 9.0f;                     // a row's reference follows its maximum when that is 2^kRise above it
// Registers per thread of the softmax, conversion and loading/issuing warpgroups: 4·96 + 2·40 + 40 = 504, what the CTA is
// launched with (7·72).
constexpr int kLaunchRegs = 72, kSoftmaxRegs = 96, kConvRegs = 40, kMiscRegs = 40;
static_assert(4 * kSoftmaxRegs + 2 * kConvRegs + kMiscRegs <= 7 * kLaunchRegs, "more registers than the launch holds");
static_assert(kTcThreads == 7 * 128 && kTcThreads * kLaunchRegs <= 65536, "one CTA's registers");
// Named barriers (0 is __syncthreads)
constexpr int kBarIssue = 2;   // + query tile: softmax warps with rows arrive, the issuing warp waits (Q or P is in TMEM)
constexpr int kBarTurn = 12;   // + query tile: a group waits for its turn, the other arrives
constexpr int kBarConv = 14;   // + 1 for V: conversion warps
constexpr int kBarJoin = 4;    // both groups, at the end of split items
constexpr int kBarEnd = 5;     // + query tile: end of an item
constexpr int kBarPair = 8;    // + 2 query tile + quadrant / 2: the warps that share rows, of two quadrants
// A tile of 128 rows: eight rows take 2 KB, raw (64 fp32 each) or split (64 fp16 of hi each, then of lo).
constexpr uint32_t kGroup = 2048, kLo = 1024, kTile = 16 * kGroup;
constexpr int kTcPart = 2 * kTcRows * (kTcDim + 2);  // floats of one partial result
// TMEM columns: S and P of both query tiles, their P·V, their Q (hi, lo: 32 columns each)
__host__ __device__ constexpr uint32_t col_s(int t) { return 128u * (uint32_t)t; }
__host__ __device__ constexpr uint32_t col_pv(int t) { return 256u + 64u * (uint32_t)t; }
__host__ __device__ constexpr uint32_t col_q(int t) { return 384u + 64u * (uint32_t)t; }

// One run of key tiles [t0, t1) of 256 query rows of a (request, kv head).
struct Item {
  int req, first, shift, len;  // first row of the request, position of its first new token, keys
  int kvh, row0, rows;         // first query row of the item, query rows of the kv head
  int t0, t1, end[2];          // key tiles, and where they end for each query tile (causality; t0 if it has no rows)
  int split;                   // one query tile, whose key tiles the two softmax groups share out
  int whole, c0, c1;           // 1 if these are all key tiles of the rows; the CTAs that share them
  int stop;                    // no further item
};

struct TcShared {
  uint64_t raw[2][kTcStages];    // [K, V]: the raw tile has landed
  uint64_t conv[2][kTcStages];   // it is split
  uint64_t empty[2][kTcStages];  // both query tiles' products have read it
  uint64_t s_full[2], pv_full[2], drained[2];  // per query tile
  uint64_t item_full[kItems], item_free[kItems];
  Item items[kItems];
  int64_t tmp[2 * kTcThreads / 32];
  int64_t off;
  alignas(16) uint32_t seen[2][kTcRing][4];  // [K, V]: keys of a tile that exist and that its scale suits (bit per key)
  float row_x[2][2][kTcRows];    // [query tile][half]: what the two threads of a row exchange
  float row_top[2][2][2][kTcRows];  // [turn][query tile][half]: their largest scores of a key tile, two sets
  alignas(16) uint32_t range[2][2][kConvWarps];  // converter warps' largest numbers and smallest pairs, as bf16 bits
  uint2 columns[2][kConvWarps][16];              // ... largest number of each head dim, four to a group
  uint32_t keys[2][kTcKeys];                     // a key's (a value's) largest group, and kSound
  uint32_t small[kTcRing][4];                    // values left out of a tile that are smaller than the others
  float k_sorted[2 * kSoftmaxWarps];             // of a softmax warp: K's scale above which a sorted tile may be fp32 work
  alignas(16) float v_scale[kTcRing][kTcDim];    // of a sorted V tile: `scale` for each head dim
  float join_m[kTcRows], join_l[kTcRows];        // split items: the second group's maxima and sums
  // what a product with the tile is multiplied by to undo the tile's scale; negative: the tile was sorted, and keys may be left
  // to the fp32 path
  float scale[2][kTcRing];
  int req;
  int unplaced;                  // a row range is invalid
  volatile int abort;
  int last[2];
  uint32_t tmem;
};
constexpr int kTcSmem = 1024 + 2 * kTcStages * (int)kTile + (int)sizeof(TcShared);

// kind::f16 descriptors: fp16 operands, fp32 accumulator; b_mn: B stored with its N index contiguous.
__host__ __device__ constexpr uint32_t idesc_f16(int m, int n, bool b_mn) {
  return (1u << 4) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// Shared-memory descriptor of hi (or, kLo further, of lo): SWIZZLE_128B, groups of eight rows kGroup apart.
__device__ __forceinline__ uint64_t desc_split(uint32_t addr) {
  return (uint64_t)((addr & 0x3FFFF) >> 4) | (uint64_t)1 << 16 | (uint64_t)(kGroup >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

// D (TMEM) (+)= A (TMEM, two fp16 per column) · B (shared), issued by the lane whose `leader` is set. The whole warp runs
// the surrounding code, so addresses and descriptors stay in uniform registers (from a branch of one lane each product
// took about 100 cycles to issue).
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc), "r"(leader));
}
__device__ __forceinline__ void commit_if(uint64_t* bar, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
      "r"(leader)
      : "memory");
}

// Bounded wait that also gives up once another role of the CTA has (abort may be null). Each try suspends the thread up
// to kSuspendNs or until the phase completes: without the hint a try returned at once so often that the waiting warps'
// polls were half of all instructions issued.
constexpr uint32_t kSuspendNs = 20000, kTries = 1u << 18;
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, volatile int* abort) {
  const uint32_t addr = smem_u32(bar);
#pragma unroll 1
  for (uint32_t i = 0; i < kTries; i++) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(addr), "r"(parity), "r"(kSuspendNs)
        : "memory");
    if (done) return true;
    if (abort && *abort) return false;
  }
  if (abort) *abort = 1;
  return false;
}
// The whole warp polls (a poll by one lane and a shuffle take twice the 150 cycles of this).
__device__ __forceinline__ bool warp_wait_bar(uint64_t* bar, uint32_t parity, volatile int* abort) {
  const bool ok = wait_bar(bar, parity, abort);
  return __all_sync(0xffffffffu, ok);
}
// Named barriers. A warp meets them as a whole, whatever branch one of its lanes has just taken.
__device__ __forceinline__ void bar_named(int id, int threads) {
  __syncwarp();
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
__device__ __forceinline__ void bar_signal(int id, int threads) {
  __syncwarp();
  asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// A query row's scale times a key tile's, above which scores could be some thousand (numbers of the two up to 2^12 in product):
// made once by the tensor cores and once in fp32 they could differ by more than 1. Weights of both kinds would no longer go
// together for a value that is left out, so all of such a tile is fp32 work then.
constexpr float kMostScore = 1.52587890625e-5f;  // 2^-16
// The power of two that brings a magnitude (bits of a finite fp32, sign cleared) to [2^13, 2^14), and its inverse.
// Magnitudes under 2^-112 keep the largest scale.
__device__ __forceinline__ void tile_scale(uint32_t bits, float& up, float& down) {
  const int e = max(14, (int)(bits >> 23));  // biased exponent
  up = __uint_as_float((uint32_t)(267 - e) << 23);
  down = __uint_as_float((uint32_t)(e - 13) << 23);
}
__device__ __forceinline__ bool finite_bits(uint32_t bits) { return bits < 0x7f800000u; }
// Magnitudes as bf16 bits (16 bits, exponent in steps of kExp): one lies more than 2^kApartExp below another.
constexpr uint32_t kExp = 128, kApartExp = 16, kApart = kApartExp * kExp;
// 2^e x, for x a power of two; 0 below the normal numbers. e x is no larger than they are.
__device__ __forceinline__ float times_pow2(float x, int e) {
  const int field = (int)(__float_as_uint(x) >> 23) + e;
  return field > 0 ? __uint_as_float((uint32_t)field << 23) : 0.0f;
}

constexpr uint32_t kInf = 255 * kExp, kTiny = 67 * kExp, kUnit = 140 * kExp;  // infinity, 2^-60, what has a scale of 1
// max(|x|, |z|) and max(|y|, |w|) of four numbers, rounded to bf16; NaN counts as the largest.
__device__ __forceinline__ __nv_bfloat162 max_abs4(float4 f) {
  return __hmax2_nan(__habs2(__floats2bfloat162_rn(f.x, f.y)), __habs2(__floats2bfloat162_rn(f.z, f.w)));
}
__device__ __forceinline__ uint32_t bits2(__nv_bfloat162 x) { return *reinterpret_cast<const uint32_t*>(&x); }

__device__ __forceinline__ uint32_t pack2(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
// Two fp32 numbers as fp16 hi parts and fp16 remainders (first number in the low half).
__device__ __forceinline__ void split2(float2 x, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __float22half2_rn(x);
  const float2 f = __half22float2(h);
  hi = pack2(h);
  lo = pack2(__float22half2_rn(__ffma2_rn(f, make_float2(-1.0f, -1.0f), x)));
}

// A request's units: per kv head, groups of 256 rows, each with the key tiles that its last row attends. A tile counts as
// many units as it takes time, about 8,400 cycles for two query tiles, 5,300 for one (chunks among decoding requests 129 us,
// 145 when all count alike), unless there are so few that a CTA has no more than two: then each counts alike, so that more
// CTAs have one (small heads, 131 new tokens of 5 requests: 26.8 us, 28.2 with weights).
struct Weights {
  int one, two;  // units of a key tile of a group of one, of two query tiles
  __device__ __forceinline__ int of(int rows, int group) const { return rows - group * 2 * kTcRows > kTcRows ? two : one; }
};
struct Shape {
  int rows, groups;   // per kv head
  int64_t ones, twos;  // key tiles of one kv head's groups of one and of two query tiles
  __device__ __forceinline__ int64_t units(const Weights& w) const { return ones * w.one + twos * w.two; }
};
__device__ __forceinline__ int group_tiles(const AttnArgs& a, const Req& r, int rows, int group) {
  const int last = min(rows, (group + 1) * 2 * kTcRows) - 1;
  const int keys = r.len - r.n + a.heads.div(last) + 1;  // that the group's last row attends
  return max(1, (keys + kTcKeys - 1) / kTcKeys);
}
__device__ __forceinline__ Shape shape_of(const AttnArgs& a, const Req& r) {
  Shape s;
  s.rows = r.n * a.g;
  s.groups = (s.rows + 2 * kTcRows - 1) / (2 * kTcRows);
  s.ones = s.twos = 0;
#pragma unroll 1
  for (int i = 0; i < s.groups; i++) (i + 1 < s.groups || s.rows - i * 2 * kTcRows > kTcRows ? s.twos : s.ones) += group_tiles(a, r, s.rows, i);
  return s;
}

// Item i for a whole warp, in shared memory until free_item(); null when there is none. Waits the whole time limit whether
// another role gave up or not: the warps that meet at named barriers must all see an item or none.
__device__ __forceinline__ const Item* take_item(TcShared& sh, int i) {
  const int slot = i % kItems;
  if (!warp_wait_bar(&sh.item_full[slot], (i / kItems) & 1, nullptr) || sh.items[slot].stop) return nullptr;
  return &sh.items[slot];
}
__device__ __forceinline__ void free_item(TcShared& sh, int i) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(&sh.item_free[i % kItems]);
}

// ---------------------------------------------------------------- roles
// Of a row's groups of four: how many are within 2^16 of its largest number (in bf16 bits), in the upper half, and how many
// further below but not 0. A call that reads the row again, as what it holds would be taken from all of the softmax.
__device__ __noinline__ uint32_t row_groups(const float* q, int dims, float scale_hi, float scale_lo, uint32_t largest) {
  uint32_t near = 0, far = 0;
#pragma unroll 1
  for (int d = 0; d < dims; d += 4) {
    uint32_t four = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const uint32_t b = __float_as_uint(fmaf(q[d + e], scale_hi, q[d + e] * scale_lo)) & 0x7fffffffu;
      if (finite_bits(b)) four = max(four, b);
    }
    if (four != 0) ((four >> 16) + kApart >= largest ? near : far)++;
  }
  return near << 16 | far;
}

// Softmax of query tile `tile`. After a timed-out wait `ok` stays false: no further TMEM or barrier-object work, but the
// named barriers are met.
__device__ __forceinline__ void softmax_role(const AttnArgs& a, TcShared& sh, uint32_t tmem) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = warp & 3, tile = warp >> 3, half = (warp >> 2) & 1;
  const int row = quad * 32 + lane;
  const uint32_t base = tmem + ((uint32_t)(quad * 32) << 16);
  const uint32_t cs = base + col_s(tile) + 64 * half, cpv = base + col_pv(tile) + 32 * half, cq = base + col_q(tile) + 16 * half;
  const int pair = kBarPair + 2 * tile + (quad >> 1), end_bar = kBarEnd + tile;
  bool ok = true;
  int J = 0, C = 0;  // key tiles of the CTA and of this query tile so far
  int pair_threads = 0;
  // The other thread's value of this row.
  auto exchange = [&](float v) {
    bar_named(pair, pair_threads);  // the last value has been read
    sh.row_x[tile][half][row] = v;
    bar_named(pair, pair_threads);
    return sh.row_x[tile][half ^ 1][row];
  };
  const Item* p_it;
  for (int i = 0; (p_it = take_item(sh, i)) != nullptr; free_item(sh, i), i++) {
    const Item& it = *p_it;
    const int first = it.row0 + (it.split ? 0 : tile * kTcRows);
    if (first >= it.rows) {
      J += it.t1 - it.t0;
      continue;
    }
    const int step = it.split ? 2 : 1, t0 = it.t0 + (it.split ? tile : 0);
    const int end = t0 + (max(0, (tile == 0 ? it.end[0] : it.end[1]) - t0) + step - 1) / step * step;
    const int quads = min(4, (it.rows - first + 31) >> 5);  // quadrants of this group that have rows
    // The groups take turns at the softmax, so that each runs beside the other's products: the x-th of the first group,
    // the x-th of the second, the x+1-th of the first, for the `turns` that both have. Left alone they fall into step,
    // wait for the tensor cores together and then compute together. Each signal is waited for once, the second group's
    // last one by the first before it leaves the item, so that no group signals twice before it is heard.
    const int first1 = it.row0 + (it.split ? 0 : kTcRows);
    const int both = 64 * (min(4, (it.rows - it.row0 + 31) >> 5) + max(0, min(4, (it.rows - first1 + 31) >> 5)));
    const int other = first1 >= it.rows ? 0 : it.split ? (it.end[0] - it.t0 + tile) >> 1 : (tile ? it.end[0] : it.end[1]) - it.t0;
    const int mine = (end - t0) / step, turns = min(mine, other);
    if (quad >= quads) {
      // None of this warp's rows exists. What is left in its rows of TMEM goes into no other row.
      J += it.t1 - it.t0;
      C += (end - t0) / step;
      bar_named(end_bar, 256 + 32);
      if (it.split) {
        bar_named(kBarJoin, 512);
        bar_named(kBarJoin, 512);
      }
      if (!it.whole && !(it.split && tile == 1)) {
        bar_named(end_bar, 256);
        bar_named(end_bar, 256);
      }
      continue;
    }
    pair_threads = 64 * min(2, quads - (quad & 2));
    const int r = first + row;
    const bool live = r < it.rows;
    const int s = a.heads.div(r), h = it.kvh * a.g + (r - s * a.g);
    const int limit = live ? it.shift + s : -1;  // the last key this row attends
    const int first_limit = it.shift + a.heads.div(first);
    // What undoes the row's scale; and K's scale above which a tile may be fp32 work for the warp, for sorted tiles in sh.k_sorted.
    // They are 0 if it is, because numbers of a row lie too far apart: where more than half of its groups are far below the
    // largest, whatever the keys; where half are or are 0, with keys of a sorted tile, of which also half of the groups count.
    // (Where fewer are, row and key share groups that count, and products of the others are small beside those.)
    float qdown, k_most;
    {
      const float* p = a.q + (int64_t)(it.first + s) * a.q0 + (int64_t)h * a.q1;
      float x[32];
#pragma unroll
      for (int d = 0; d < 32; d += 4) {
        float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
        if (live && 32 * half + d < a.D) {  // the head dim is a multiple of 4
          const float* q = p + 32 * half + d;
          if (a.q_vec) f = *reinterpret_cast<const float4*>(q);
          else f = make_float4(q[0], q[1], q[2], q[3]);
        }
        x[d] = f.x; x[d + 1] = f.y; x[d + 2] = f.z; x[d + 3] = f.w;
      }
      uint32_t big = 0, least = 0xffffffffu;  // largest number, smallest of the groups of four
#pragma unroll
      for (int d = 0; d < 32; d += 4) {
        uint32_t four = 0;
#pragma unroll
        for (int e = d; e < d + 4; e++) {
          x[e] = fmaf(x[e], a.scale_hi, x[e] * a.scale_lo);  // scores in powers of two
          const uint32_t b = __float_as_uint(x[e]) & 0x7fffffffu;
          if (finite_bits(b)) four = max(four, b);
        }
        big = max(big, four);
        if (32 * half + d < a.D) least = min(least, four);
      }
      // both in one word, in 16 bits each: the scale needs no more than the exponent
      const uint32_t theirs = __float_as_uint(exchange(__uint_as_float((big & 0xffff0000u) | (least >> 16))));
      big = max(big, theirs & 0xffff0000u);
      least = min(least >> 16, theirs & 0xffffu);
      float up;
      tile_scale(big, up, qdown);
      k_most = kMostScore / __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(qdown)));
      const bool uneven = __any_sync(0xffffffffu, least + kApart < (big >> 16));
#pragma unroll
      for (int c = 0; c < 2; c++) {  // 16 elements: 8 columns of hi, 8 of lo
        float hi[8], lo[8];
#pragma unroll
        for (int d = 0; d < 8; d++) {
          uint32_t h, l;
          split2(make_float2(x[16 * c + 2 * d] * up, x[16 * c + 2 * d + 1] * up), h, l);
          hi[d] = __uint_as_float(h);
          lo[d] = __uint_as_float(l);
        }
        tc::tmem_st8(cq + 8 * c, hi);
        tc::tmem_st8(cq + 32 + 8 * c, lo);
      }
      tmem_st_wait();
      fence_before();
      bar_signal(kBarIssue + tile, 64 * quads + 32);
      float k_sorted = k_most;
      if (uneven) {
        const uint32_t groups = row_groups(p, live ? a.D : 0, a.scale_hi, a.scale_lo, big >> 16);
        __syncwarp();
        if (__any_sync(0xffffffffu, big != 0 && 8 * (groups >> 16) <= (uint32_t)a.D)) k_sorted = 0.0f;
        if (__any_sync(0xffffffffu, 8 * (groups & 0xffffu) > (uint32_t)a.D)) k_most = 0.0f;
      }
      if (lane == 0) sh.k_sorted[warp] = k_sorted;
      __syncwarp();
    }
    float2 o[16];
#pragma unroll
    for (int d = 0; d < 16; d++) o[d] = make_float2(0.0f, 0.0f);
    float m = -INFINITY, l = 0.0f;  // reference and sum of the weights
#pragma unroll 1
    for (int t = t0; t < end; t += step) {
      const int j = J + t - it.t0, slot = j % kTcRing, turn = (t - t0) / step;
      if (ok && !warp_wait_bar(&sh.s_full[tile], C & 1, &sh.abort)) ok = false;
      if (tile == 0 ? turn > 0 && turn <= turns : turn < turns) bar_named(kBarTurn + tile, both);
      fence_after();
      // kept finite and above 0: a score of 0 or -inf times it stays one
      const float kdown = sh.scale[0][slot];
      const float c = fminf(fmaxf(fabsf(qdown * kdown), 1.1754944e-38f), 3.4028235e38f);
      bool all_fp32 = __float_as_uint(kdown) > __float_as_uint(k_most);  // or the tile is sorted
      const uint4 seen = *reinterpret_cast<const uint4*>(sh.seen[0][slot]);
      if (t * kTcKeys + kTcKeys - 1 > first_limit || (seen.x & seen.y & seen.z & seen.w) != 0xffffffffu || all_fp32) {
        if (all_fp32) {
          const float least = kdown > 0.0f ? k_most : sh.k_sorted[warp];
          all_fp32 = fabsf(kdown) > least;
          if (all_fp32 && least > 0.0f) {  // only where values are left out; V cannot be split anew before this P
            if (ok && !warp_wait_bar(&sh.conv[1][j % kTcStages], (j / kTcStages) & 1, &sh.abort)) ok = false;
            all_fp32 = sh.scale[1][slot] < 0.0f;
          }
        }
        // scores of keys that do not exist or that the row does not attend become -inf in place
#pragma unroll 1
        for (int g = 0; g < 4; g++) {
          const int k0 = 64 * half + 16 * g, n = all_fp32 ? 0 : limit - (t * kTcKeys + k0) + 1;
          const uint32_t vis = (sh.seen[0][slot][k0 >> 5] >> (k0 & 31)) & (n >= 16 ? 0xffffu : n <= 0 ? 0u : (1u << n) - 1u);
          float x[16];
          tc::tmem_ld16(cs + 16 * g, x);
#pragma unroll
          for (int e = 0; e < 16; e++) x[e] = (vis >> e) & 1u ? x[e] : -INFINITY;
          tc::tmem_st16(cs + 16 * g, x);
        }
        tmem_st_wait();
      }
      float top = -INFINITY;
#pragma unroll 1
      for (int g = 0; g < 2; g++) {
        float x[32], y = -INFINITY;
        tmem_ld32(cs + 32 * g, x);
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          top = fmaxf(top, fmaxf(x[e], x[e + 1]));
          y = fmaxf(y, fmaxf(x[e + 2], x[e + 3]));
        }
        top = fmaxf(top, y);
      }
      float* tops = sh.row_top[C & 1][tile][0];  // two sets: the one before may still be read
      top *= c;  // a power of two
      tops[half * kTcRows + row] = top;
      bar_named(pair, pair_threads);
      top = ceilf(fmaxf(top, tops[(half ^ 1) * kTcRows + row]));
      // rounded down, so that no weight is above 2^14, however large the scores: fp16 holds none of 2^16
      const float ref = __fsub_rd(14.0f, top == -INFINITY ? 0.0f : top);
      const float2 c2 = make_float2(c, c), ref2 = make_float2(ref, ref);
      float2 sum0 = make_float2(0.0f, 0.0f), sum1 = sum0;
#pragma unroll 1
      for (int g = 0; g < 4; g++) {
        float x[16], w[16];
        tc::tmem_ld16(cs + 16 * g, x);
#pragma unroll
        for (int e = 0; e < 8; e++) {
          float2 p = __ffma2_rn(make_float2(x[2 * e], x[2 * e + 1]), c2, ref2);
          p.x = ex2_sfu(p.x);
          p.y = ex2_sfu(p.y);
          if (e & 1) sum1 = __fadd2_rn(sum1, p);
          else sum0 = __fadd2_rn(sum0, p);
          uint32_t hi, lo;
          split2(p, hi, lo);
          w[e] = __uint_as_float(hi);
          w[8 + e] = __uint_as_float(lo);
        }
        tc::tmem_st16(cs + 16 * g, w);  // over the scores just read: 16 keys as 8 columns of hi, 8 of lo
      }
      tmem_st_wait();
      fence_before();
      bar_signal(kBarIssue + tile, 64 * quads + 32);
      if (turn < turns) bar_signal(kBarTurn + (tile ^ 1), both);
      const bool rise = top > m + kRise;  // also from -inf, never on NaN
      if (__any_sync(0xffffffffu, rise)) {
        const float alpha = rise ? times_pow2(1.0f, (int)fmaxf(m - top, -1000.0f)) : 1.0f;
        if (rise) m = top;
        const float2 al = make_float2(alpha, alpha);
        l *= alpha;
#pragma unroll
        for (int d = 0; d < 16; d++) o[d] = __fmul2_rn(o[d], al);
      }
      // from the tile's weights, against -ref, to the row's, against m + kRise
      const int shift = (int)fmaxf(top == -INFINITY ? -1000.0f : -ref - m, -1000.0f) - (int)kRise;
      l = fmaf((sum0.x + sum0.y) + (sum1.x + sum1.y), times_pow2(1.0f, shift), l);
      if (ok && !warp_wait_bar(&sh.pv_full[tile], C & 1, &sh.abort)) ok = false;
      C++;
      fence_after();
      const float vdown = sh.scale[1][slot];
      if (fminf(kdown, vdown) < 0.0f || all_fp32) {
        // Keys that are left to fp32: those that sh.seen misses, or all where a row of q has its numbers too far apart. One at a
        // time, and what can be made again is: registers are taken from the loop around (four prompt chunks of 2,000 653 us;
        // with four keys at a time 746).
        // pass 0: the largest score of keys whose values are small ones left out; pass 1: values left out; pass 2: keys left
        // out. Where a small value has the largest weight of the tile, the others, taken against that, may have lost what
        // counts beside it: then pass 1 takes all values of the tile, and P·V is not used.
        int my_row = r, my_slot = slot, key0 = t * kTcKeys, my_half = half;
        asm volatile("" : "+r"(my_row), "+r"(my_slot), "+r"(key0), "+r"(my_half));  // none of this is made ahead of the branch
        const bool all = all_fp32, v_drops = !all && vdown < 0.0f;
        bool near = false;
#pragma unroll 1
        for (int pass = !ok ? 3 : v_drops ? 0 : 2; pass < 3; pass++) {
          if (pass == 1) near = __any_sync(0xffffffffu, near);
          if (!all && !near && pass == (v_drops ? 1 : 2)) {
            const float f = times_pow2(1.0f, shift);
#pragma unroll
            for (int d = 0; d < 16; d += 4) {
              float x[8];
              tc::tmem_ld8(cpv + 2 * d, x);
#pragma unroll
              for (int e = 0; e < 4; e++) {
                float2 down = make_float2(vdown, vdown);
                if (vdown < 0.0f) down = *reinterpret_cast<const float2*>(&sh.v_scale[my_slot][32 * my_half + 2 * (d + e)]);
                o[d + e] = __ffma2_rn(__fmul2_rn(make_float2(x[2 * e], x[2 * e + 1]), make_float2(f, f)), down, o[d + e]);
              }
            }
          }
#pragma unroll 1
          for (int k = 0; k < kTcKeys; k++) {
            const uint32_t k_fits = sh.seen[0][my_slot][k >> 5];
            uint32_t take = ~0u;
            if (!all) {
              if (pass == 0) take = k_fits & sh.small[my_slot][k >> 5];
              else if (pass == 1) take = near ? k_fits : k_fits & ~sh.seen[1][my_slot][k >> 5];
              else take = ~k_fits;
            }
            take >>= k & 31;
            if (take == 0) k |= 31;  // none in the rest of the word
            if (!(take & 1u)) continue;
            const int pi = a.page.div(key0 + k);
            int page;
            if (key0 + k >= it.len) continue;
            if (!integral(a.table[(int64_t)it.req * a.t0 + pi * a.t1], 0, a.pages - 1, page)) continue;
            const int64_t at = (int64_t)page * a.c0 + (int64_t)it.kvh * a.c1 + (int64_t)(key0 + k - pi * a.page.size) * a.c2;
            const int rr = min(my_row, it.rows - 1), sr = a.heads.div(rr);
            const float* q = a.q + (int64_t)(it.first + sr) * a.q0 + (int64_t)(it.kvh * a.g + (rr - sr * a.g)) * a.q1;
            const bool on = my_row < it.rows && key0 + k <= it.shift + sr;  // the row attends it
            float x = 0.0f;
#pragma unroll 1
            for (int d = 0; d < a.D; d += 4) {
              const float4 f = a.q_vec ? *reinterpret_cast<const float4*>(q + d)
                                       : make_float4(q[d], q[d + 1], q[d + 2], q[d + 3]);
              const float4 y = *reinterpret_cast<const float4*>(a.k + at + d);
              x = fmaf(fmaf(f.x, a.scale_hi, f.x * a.scale_lo), y.x, x);
              x = fmaf(fmaf(f.y, a.scale_hi, f.y * a.scale_lo), y.y, x);
              x = fmaf(fmaf(f.z, a.scale_hi, f.z * a.scale_lo), y.z, x);
              x = fmaf(fmaf(f.w, a.scale_hi, f.w * a.scale_lo), y.w, x);
            }
            if (pass == 0) {
              near = near || (on && x > top - 1.0f);
              continue;
            }
            if (pass == 2 && on && ceilf(x) > m + kRise) {
              const float alpha = times_pow2(1.0f, (int)fmaxf(m - ceilf(x), -1000.0f));
              m = ceilf(x);
              l *= alpha;
#pragma unroll
              for (int d = 0; d < 16; d++) o[d] = __fmul2_rn(o[d], make_float2(alpha, alpha));
            }
            if (on) {  // a value that the row does not attend may be anything: it is left out, not multiplied by 0
              const float w = ex2_sfu(x - (m == -INFINITY ? 0.0f : m) - kRise);  // m + kRise may round to m
              if (pass == 2 && my_half == 0) l += w;  // the sums of both halves are joined
              const float* v = a.v + at + 32 * my_half;
#pragma unroll
              for (int d = 0; d < 8; d++) {
                if (32 * my_half + 4 * d >= a.D) break;
                const float4 y = *reinterpret_cast<const float4*>(v + 4 * d);
                o[2 * d] = __ffma2_rn(make_float2(y.x, y.y), make_float2(w, w), o[2 * d]);
                o[2 * d + 1] = __ffma2_rn(make_float2(y.z, y.w), make_float2(w, w), o[2 * d + 1]);
              }
            }
            __syncwarp();
          }
        }
      } else {
        const float down = times_pow2(vdown, shift);
        const float2 f = make_float2(down, down);
#pragma unroll
        for (int c = 0; c < 2; c++) {
          float x[16];
          tc::tmem_ld16(cpv + 16 * c, x);
#pragma unroll
          for (int d = 0; d < 8; d++) o[8 * c + d] = __ffma2_rn(make_float2(x[2 * d], x[2 * d + 1]), f, o[8 * c + d]);
        }
      }
    }
    if (tile == 0 && turns > 0 && mine == turns) bar_named(kBarTurn, both);
    l += exchange(l);  // before the group meets: the next item's rows may pair its warps differently
    // Every warp has read the last scales before the issuing warp frees tiles that the ring's slots are reused for, and
    // none of this group, those without rows included, gets ahead to the next item's barriers.
    bar_named(end_bar, 256 + 32);
    J += it.t1 - it.t0;
    if (it.split) {
      // The second group's result goes to the first through the second's P·V columns (free until its next P).
      if (tile == 1 && ok) {
        tmem_st32(cpv, reinterpret_cast<const float*>(o));
        tmem_st_wait();
        fence_before();
        sh.join_m[row] = m;
        sh.join_l[row] = l;
      }
      bar_named(kBarJoin, 512);
      if (tile == 0 && ok) {
        fence_after();
        const float m1 = sh.join_m[row], mn = fmaxf(m, m1);
        const float f0 = mn == m ? 1.0f : ex2_sfu(m - mn), f1 = mn == m1 ? 1.0f : ex2_sfu(m1 - mn);
        m = mn;
        l = l * f0 + sh.join_l[row] * f1;
        const float2 g0 = make_float2(f0, f0), g1 = make_float2(f1, f1);
        float x[32];
        tmem_ld32(base + col_pv(1) + 32 * half, x);
#pragma unroll
        for (int d = 0; d < 16; d++) o[d] = __ffma2_rn(make_float2(x[2 * d], x[2 * d + 1]), g1, __fmul2_rn(o[d], g0));
        fence_before();
      }
      bar_named(kBarJoin, 512);
      if (tile == 1) continue;
    }
    bool write = it.whole != 0;
    if (!write) {
      const int c0 = it.c0, c1 = it.c1;
      // a row's pairs of head dims kTcRows apart, so that a warp's 32 rows lie side by side; then its (m, l)
      auto part_of = [&](int b) {
        return reinterpret_cast<float2*>(a.part + (size_t)(2 * b + (b == c0 ? 1 : 0)) * kTcPart + (size_t)tile * (kTcPart / 2)) + row;
      };
      float2* mine = part_of(blockIdx.x);
#pragma unroll
      for (int d = 0; d < 16; d++) mine[(16 * half + d) * kTcRows] = o[d];
      if (half == 0) mine[32 * kTcRows] = make_float2(m, l);
      __threadfence();
      bar_named(end_bar, 256);
      if (row == 0 && half == 0) {
        unsigned* ticket = &a.tickets[2 * c0 + tile];
        sh.last[tile] = atomicAdd(ticket, 1u) == (unsigned)(c1 - c0);
        if (sh.last[tile]) *ticket = 0;
      }
      bar_named(end_bar, 256);
      write = sh.last[tile] != 0;
      if (write) {
        __threadfence();
        // one pass: the sums so far move to a larger reference when one comes
        float2 ml = __ldcg(part_of(c0) + 32 * kTcRows);
        m = -INFINITY;
        l = 0.0f;
#pragma unroll
        for (int d = 0; d < 16; d++) o[d] = make_float2(0.0f, 0.0f);
#pragma unroll 1
        for (int b = c0; b <= c1; b++) {
          const float2* p = part_of(b);
          float2 x[16];
#pragma unroll
          for (int d = 0; d < 16; d++) x[d] = __ldcg(p + (16 * half + d) * kTcRows);
          const float2 now = ml;
          if (b < c1) ml = __ldcg(part_of(b + 1) + 32 * kTcRows);
          const float mn = fmaxf(m, now.x);
          const float f0 = mn == m ? 1.0f : ex2_sfu(m - mn), f1 = mn == now.x ? 1.0f : ex2_sfu(now.x - mn);
          m = mn;
          l = l * f0 + now.y * f1;
          const float2 g0 = make_float2(f0, f0), g1 = make_float2(f1, f1);
#pragma unroll
          for (int d = 0; d < 16; d++) o[d] = __ffma2_rn(x[d], g1, __fmul2_rn(o[d], g0));
        }
      }
    }
    if (write && ok && live) {
      float* out = a.out + ((int64_t)(it.first + s) * a.H + h) * a.D + 32 * half;
      const float inv = 1.0f / l;
#pragma unroll
      for (int d = 0; d < 8; d++)
        if (32 * half + 4 * d < a.D)
          *reinterpret_cast<float4*>(out + 4 * d) =
              l == 0.0f ? make_float4(0.f, 0.f, 0.f, 0.f)
                        : make_float4(o[2 * d].x * inv, o[2 * d].y * inv, o[2 * d + 1].x * inv, o[2 * d + 1].y * inv);
    }
  }
  if (!ok && lane == 0) {
    atomicExch(a.error_flag, 76);
    sh.abort = 1;
  }
}

// For a tile whose numbers lie far apart: finds the scale that suits most keys, takes the others out of sh.seen and makes them
// 0. Returns the magnitude (in bf16 bits; 0 if there is none) that bounds the tile's numbers. V has a scale for each head dim, as
// a product's columns may be scaled as one likes, and is multiplied here. `rows` is the lane's place in its warp's rows.
//   K: a key fits if it is no larger than that, and no more than 2^16 smaller, nor are half of its groups (a few head dims that
//      are always small cost nothing; one that is always large would cost the others their precision);
//   V: a value fits if its largest number is, and if then none of its groups is all 2^16 below the others that fit: weights are
//      taken against the largest, which may be its own, and lose what is further below.
// A call: in place it costs the loop around it 2% (six new tokens of 16 requests).
constexpr uint32_t kNeutral = 1u << 31;  // the key does not count
__device__ __noinline__ uint32_t sort_keys(TcShared& sh, uint8_t* rows, int dims, int op, int slot, bool ok) {
  const int warp = (threadIdx.x >> 5) & 3, lane = threadIdx.x & 31, tr = lane >> 4, tc4 = lane & 15;
  const uint32_t seen = ok ? sh.seen[op][slot][warp] : 0u;
  uint32_t* keys = sh.keys[op];
  auto group = [&](int e) {  // the lane's four numbers of row 2 e + tr
    const float4 f = *reinterpret_cast<const float4*>(rows + e * 512);
    const __nv_bfloat162 a = __floats2bfloat162_rn(f.x, f.y), b = __floats2bfloat162_rn(f.z, f.w);
    return make_uint2(bits2(a) & 0x7fff7fffu, bits2(b) & 0x7fff7fffu);
  };
  auto most = [](uint2 g) { return max(max(g.x & 0xffffu, g.x >> 16), max(g.y & 0xffffu, g.y >> 16)); };
  auto larger = [](uint2 a, uint2 b) { return make_uint2(__vmaxu2(a.x, b.x), __vmaxu2(a.y, b.y)); };
  // the largest of the lane's head dims in those of the warp's rows, and then of all rows
  auto column = [&](uint32_t of) {
    uint2 m = make_uint2(0, 0);
#pragma unroll 1
    for (int e = 0; e < 16; e++)
      if ((of >> (2 * e + tr)) & 1u) m = larger(m, group(e));
    __syncwarp();
    m = larger(m, make_uint2(__shfl_xor_sync(0xffffffffu, m.x, 16), __shfl_xor_sync(0xffffffffu, m.y, 16)));
    if (tr == 0) sh.columns[op][warp][tc4] = 4 * tc4 < dims ? m : make_uint2(0, 0);
    bar_named(kBarConv + op, 32 * kConvWarps);
    m = make_uint2(0, 0);
#pragma unroll 1
    for (int w = 0; w < kConvWarps; w++) m = larger(m, sh.columns[op][w][tc4]);
    return m;
  };
  uint2 largest = column(seen);
  const bool counts = (largest.x | largest.y) != 0;
  const int half = (dims / 4 + 1) / 2;  // of the groups
#pragma unroll 1
  for (int e = 0; e < 16; e++) {
    const bool exists = (seen >> (2 * e + tr)) & 1u;
    uint32_t hi = exists && counts ? most(group(e)) : 0;
#pragma unroll 1
    for (int o = 1; o < 16; o <<= 1) hi = max(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    if (tc4 == 0) keys[32 * warp + 2 * e + tr] = !exists || (op == 0 && hi == 0) ? kNeutral : hi;
  }
  bar_named(kBarConv + op, 32 * kConvWarps);
  auto fits = [&](uint32_t key, uint32_t top) { return key == kNeutral || (key <= top && key + kApart >= top); };
  // how many keys fit, and under which magnitude, one of the keys' own: the largest if all do
  uint32_t best = 0, count = 0;
#pragma unroll 1
  for (int c = lane; c < kTcKeys; c += 32)
    if (keys[c] < kInf) best = max(best, keys[c]);
  __syncwarp();
  best = __reduce_max_sync(0xffffffffu, best);
#pragma unroll 1
  for (int c = lane; c < kTcKeys; c += 32) count += fits(keys[c], best) ? 1u : 0u;
  __syncwarp();
  count = __reduce_add_sync(0xffffffffu, count);
  if (count < kTcKeys) {
    best = 0;
#pragma unroll 1
    for (int c = lane; c < kTcKeys; c += 32) {
      const uint32_t top = keys[c];
      if (top == 0 || top >= kInf) continue;
      count = 0;
#pragma unroll 1
      for (int i = 0; i < kTcKeys; i++) count += fits(keys[i], top) ? 1u : 0u;
      best = max(best, count << 16 | top);
    }
    __syncwarp();
    best = __reduce_max_sync(0xffffffffu, best) & 0xffffu;
  }
  const uint32_t key = keys[32 * warp + lane];
  uint32_t fit = __ballot_sync(0xffffffffu, best != 0 && fits(key, best)) & seen;
  uint32_t small = __ballot_sync(0xffffffffu, best == 0 || key + kApart < best) & seen & ~fit, uneven = 0;
  largest = op == 1 ? column(fit) : make_uint2(best | best << 16, best | best << 16);
#pragma unroll 1
  for (int e = 0; e < 16; e++) {
    const uint2 g = group(e);
    auto near = [&](uint32_t m, uint32_t of) { return (of != 0 && m != 0 && m + kApart >= of); };
    const bool any = near(g.x & 0xffffu, largest.x & 0xffffu) || near(g.x >> 16, largest.x >> 16) ||
                     near(g.y & 0xffffu, largest.y & 0xffffu) || near(g.y >> 16, largest.y >> 16);
    const uint32_t n = __ballot_sync(0xffffffffu, op == 1 ? (largest.x | largest.y) != 0 && !any : any);
#pragma unroll
    for (int r = 0; r < 2; r++) {
      const int of = __popc((n >> (16 * r)) & 0xffffu);
      if (op == 1 ? of > 0 : of < half && keys[32 * warp + 2 * e + r] != kNeutral) uneven |= 1u << (2 * e + r);
    }
  }
  uneven &= fit;
  fit &= ~uneven;
  small |= uneven;
  float4 up = make_float4(1.f, 1.f, 1.f, 1.f);
  if (op == 1) {
    float4 down;
    tile_scale(largest.x << 16, up.x, down.x);
    tile_scale(largest.x & 0xffff0000u, up.y, down.y);
    tile_scale(largest.y << 16, up.z, down.z);
    tile_scale(largest.y & 0xffff0000u, up.w, down.w);
    if (warp == 0 && lane < 16) *reinterpret_cast<float4*>(&sh.v_scale[slot][4 * lane]) = down;
  }
#pragma unroll 1
  for (int e = 0; e < 16; e++) {  // missing rows, too: they are copies of one that may be left out
    float4* row = reinterpret_cast<float4*>(rows + e * 512);
    float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
    if ((fit >> (2 * e + tr)) & 1u) {
      f = *row;
      f = make_float4(f.x * up.x, f.y * up.y, f.z * up.z, f.w * up.w);
    }
    *row = f;
  }
  if (lane == 0) {
    if (fit != seen) sh.seen[op][slot][warp] = fit;
    if (op == 1) sh.small[slot][warp] = small;
  }
  __syncwarp();
  return op == 1 ? kUnit : best;
}

// Splits the raw K (op 0) or V (op 1) tiles in place. A warp has four of a tile's groups of eight rows; a first pass takes
// the largest magnitude of the whole tile, a second splits group by group, so that few registers are held.
__device__ __forceinline__ void convert_role(const AttnArgs& a, TcShared& sh, uint8_t* tiles, int op) {
  const int warp = (threadIdx.x >> 5) & 3, lane = threadIdx.x & 31;
  const int tr = lane >> 4, tc4 = lane & 15;  // 16 lanes per row, two rows at a time
  // four elements of the warp's row tr (two rows are 512 bytes), and where their hi parts go: 16-byte chunk c of row r of
  // eight is stored as chunk c ^ r
  const uint32_t from = 4 * warp * kGroup + tr * 256 + 16 * tc4;
  const uint32_t to = 4 * warp * kGroup + ((tr * 128 + ((tc4 >> 1) << 4) + ((tc4 & 1) << 3)) ^ (tr << 4));
  const bool pad = 4 * tc4 >= a.D;
  bool ok = true;
  int J = 0, st = 0, parity = 0;
  const Item* p_it;
  for (int i = 0; (p_it = take_item(sh, i)) != nullptr; i++) {
    int n = p_it->t1 - p_it->t0;
    free_item(sh, i);
#pragma unroll 1
    for (; n > 0; n--) {
      uint8_t* tile = tiles + (op * kTcStages + st) * kTile;
      uint32_t big = 0, small = 0xffffu;
      if (ok && !warp_wait_bar(&sh.raw[op][st], parity, &sh.abort)) ok = false;
      if (ok) {
        const uint32_t seen = sh.seen[op][J % kTcRing][warp];  // of the warp's 32 rows
        if (seen != 0xffffffffu || a.D < kTcDim) {
          // Nothing was copied there. A missing row's weights are 0; it becomes one like the warp's first, so that it changes
          // none of what is found out below.
          float4 like = make_float4(0.f, 0.f, 0.f, 0.f);
          if (seen != 0xffffffffu && seen != 0 && !pad)
            like = *reinterpret_cast<const float4*>(tile + 4 * warp * kGroup + (__ffs(seen) - 1) * 256 + 16 * tc4);
          __syncwarp();
#pragma unroll 1
          for (int e = 0; e < 16; e++)
            if (pad || !((seen >> (2 * e + tr)) & 1u)) *reinterpret_cast<float4*>(tile + from + e * 512) = like;
        }
        // The largest magnitude, and the smallest of pairs (of a group of four), in bf16: only exponents count.
        __nv_bfloat162 most = __floats2bfloat162_rn(0.0f, 0.0f), least = __floats2bfloat162_rn(3e38f, 3e38f);
#pragma unroll 1
        for (int g = 0; g < 4; g++) {
          float4 x[4];
#pragma unroll
          for (int e = 0; e < 4; e++) x[e] = *reinterpret_cast<const float4*>(tile + from + g * kGroup + e * 512);
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const __nv_bfloat162 m = max_abs4(x[e]);
            most = __hmax2_nan(most, m);
            least = __hmin2(least, m);
          }
        }
        big = max(bits2(most) & 0xffffu, bits2(most) >> 16);
        if (!pad && seen != 0) small = min(bits2(least) & 0xffffu, bits2(least) >> 16);
      }
      const uint32_t mine = __reduce_max_sync(0xffffffffu, big) << 16 | __reduce_min_sync(0xffffffffu, small);
      uint32_t* range = sh.range[op][J & 1];  // two sets: a warp may be a tile ahead of one that still reads
      if (lane == 0) range[warp] = mine;
      bar_named(kBarConv + op, 32 * kConvWarps);
      const uint4 all = *reinterpret_cast<const uint4*>(range);
      uint32_t top = max(max(all.x, all.y), max(all.z, all.w)) >> 16;
      const uint32_t low = min(min(all.x & 0xffffu, all.y & 0xffffu), min(all.z & 0xffffu, all.w & 0xffffu));
      const bool sort = low + kApart < top || top >= kInf || (op == 1 && top != 0 && top < kTiny);
      if (sort) top = sort_keys(sh, tile + from, a.D, op, J % kTcRing, ok);
      if (ok) {
        float up, down;
        tile_scale(top << 16, up, down);
        if (warp == 0 && lane == 0) sh.scale[op][J % kTcRing] = sort ? -down : down;
        const float2 up2 = make_float2(up, up);
#pragma unroll 1
        for (int g = 0; g < 4; g++) {
          float4 x[4];
#pragma unroll
          for (int e = 0; e < 4; e++) x[e] = *reinterpret_cast<const float4*>(tile + from + g * kGroup + e * 512);
          __syncwarp();  // the group's raw rows are in registers
#pragma unroll
          for (int e = 0; e < 4; e++) {
            uint2 hi, lo;
            split2(__fmul2_rn(make_float2(x[e].x, x[e].y), up2), hi.x, lo.x);
            split2(__fmul2_rn(make_float2(x[e].z, x[e].w), up2), hi.y, lo.y);
            uint8_t* dst = tile + (to ^ (e << 5)) + g * kGroup + e * 256;
            *reinterpret_cast<uint2*>(dst) = hi;
            *reinterpret_cast<uint2*>(dst + kLo) = lo;
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.conv[op][st]);
      }
      J++;
      if (++st == kTcStages) {
        st = 0;
        parity ^= 1;
      }
    }
  }
  if (!ok && lane == 0) {
    atomicExch(a.error_flag, 77);
    sh.abort = 1;
  }
}

// 16 bytes into shared memory without a wait; the barrier's phase completes only after this lane's copies so far have.
__device__ __forceinline__ void copy16(void* to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_hold(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// Copies the raw K (op 0) or V (op 1) tiles of an item out of their pages, the CTA's tiles J and on: a page's rows with one
// bulk copy where they make 1 KB or more (a bulk copy takes some 100 cycles to issue), else 16 bytes at a time, a lane per
// row: six new tokens of 16 requests, pages of 16 positions 58 us, of 4 62; 16 bytes at a time 69 and 72. False if a wait gave up.
__device__ __forceinline__ bool load_item(const AttnArgs& a, TcShared& sh, uint8_t* tiles, int op, const Item& it, int& J,
                                          bool& bad) {
  const int lane = threadIdx.x & 31;
  const int P = a.page.size;
  const bool bulk = a.D == kTcDim && a.c2 == kTcDim && P >= 4;
  const float* trow = a.table + (int64_t)it.req * a.t0;
  const float* src = (op == 0 ? a.k : a.v) + (int64_t)it.kvh * a.c1;
  const int len = it.len, t1 = it.t1;
  // the id of the lane's page of a tile (P >= 4: one per lane at most), read a tile ahead
  auto page_id = [&](int t) -> float {
    const int pi = a.page.div(t * kTcKeys) + lane;
    return t < t1 && pi * P < min((t + 1) * kTcKeys, len) ? trow[pi * a.t1] : 0.0f;
  };
  float id = page_id(it.t0);
#pragma unroll 1
  for (int t = it.t0; t < t1; t++, J++) {
    const int st = J % kTcStages, slot = J % kTcRing;
    const int k0 = t * kTcKeys, k1 = min(k0 + kTcKeys, len);
    const int p0 = a.page.div(k0), p1 = k1 > k0 ? a.page.div(k1 - 1) : p0 - 1;
    uint32_t seen[4] = {~0u, ~0u, ~0u, ~0u};
    int to = 0;          // the lane's page's rows start at `to`,
    uint32_t bytes = 0;  // make this much
    int64_t from = 0;    // and come from this element on
    const float ahead = page_id(t + 1);
    bool whole = k1 - k0 == kTcKeys && P >= 4;
    if (P >= 4) {
      const int pi = p0 + lane, lo = max(pi * P, k0), hi = min((pi + 1) * P, k1);
      int page;
      if (pi <= p1) {
        if (integral(id, 0, a.pages - 1, page)) {
          to = lo - k0;
          bytes = (uint32_t)(hi - lo) * 256;
          from = (int64_t)page * a.c0 + (lo - pi * P) * a.c2;
        } else {
          bad = true;
          whole = false;
        }
      }
    }
    uint32_t count = kTcKeys;  // rows that exist
    if (!__all_sync(0xffffffffu, whole)) {
      count = 0;
#pragma unroll
      for (int g = 0; g < 4; g++) {
        const int j = k0 + 32 * g + lane;
        int page;
        const bool has = j < k1 && integral(trow[a.page.div(j) * a.t1], 0, a.pages - 1, page);
        if (j < k1 && !has) bad = true;
        seen[g] = __ballot_sync(0xffffffffu, has);
        count += __popc(seen[g]);
      }
    }
    id = ahead;
    if (!warp_wait_bar(&sh.empty[op][st], ((J / kTcStages) & 1) ^ 1, &sh.abort)) return false;
    uint8_t* tile = tiles + (op * kTcStages + st) * kTile;
    if (lane == 0) {
      *reinterpret_cast<uint4*>(sh.seen[op][slot]) = make_uint4(seen[0], seen[1], seen[2], seen[3]);
      if (bulk) mbar_expect_tx(&sh.raw[op][st], count * 256);
    }
    __syncwarp();
    if (bulk) {
      if (bytes > 0) bulk_g2s(tile + to * 256, src + from, bytes, &sh.raw[op][st]);
    } else {
#pragma unroll 1
      for (int j = k0 + lane; j < k1; j += 32) {
        const int pi = a.page.div(j);
        int page;
        if (!integral(trow[pi * a.t1], 0, a.pages - 1, page)) continue;
        const float* row = src + (int64_t)page * a.c0 + (int64_t)(j - pi * P) * a.c2;
        uint8_t* dst = tile + (uint32_t)(j - k0) * 256;
#pragma unroll 4
        for (int e = 0; e < a.D; e += 4) copy16(dst + 4 * e, row + e);
      }
      copies_hold(&sh.raw[op][st]);
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.raw[op][st]);
    }
  }
  return true;
}
// After the last of its J tiles: every product has signalled its stage, or at least every copy has landed, before the CTA
// may exit.
__device__ __forceinline__ void load_end(const AttnArgs& a, TcShared& sh, int op, int J, bool ok, bool bad) {
  if (bad) atomicExch(a.error_flag, 75);
  if ((threadIdx.x & 31) != 0) return;
  if (!ok) {
    atomicExch(a.error_flag, 78);
    sh.abort = 1;
  }
#pragma unroll 1
  for (int j = max(0, J - kTcStages); j < J; j++) {
    const int st = j % kTcStages;
    const uint32_t parity = (j / kTcStages) & 1;
    if (!wait_bar(&sh.empty[op][st], parity, &sh.abort)) tc::mbar_wait(&sh.raw[op][st], parity);
  }
}
__device__ __forceinline__ void load_k_role(const AttnArgs& a, TcShared& sh, uint8_t* tiles) {
  bool ok = true, bad = false;
  int J = 0;
  const Item* it;
  for (int i = 0; ok && (it = take_item(sh, i)) != nullptr; free_item(sh, i), i++) ok = load_item(a, sh, tiles, 0, *it, J, bad);
  load_end(a, sh, 0, J, ok, bad);
}

// Hands out the CTA's share of the units, [u, u1) from unit `off` of request `req` on, as items, and copies their V tiles.
// An item is published before the V tiles of the one before are copied.
__device__ __forceinline__ void walk_role(const AttnArgs& a, TcShared& sh, uint8_t* tiles, int req, int64_t off, int64_t u,
                                          int64_t u1, int64_t total, int64_t G, const Weights& weights) {
  bool ok = true, bad = false, stopped = false;
  int J = 0;
  auto publish = [&](int i) {
    if (!warp_wait_bar(&sh.item_free[i % kItems], ((i / kItems) & 1) ^ 1, &sh.abort)) {
      if ((threadIdx.x & 31) == 0) atomicExch(a.error_flag, 80);
      return false;
    }
    Item& it = sh.items[i % kItems];  // every lane writes the same
    stopped = true;
#pragma unroll 1
    while (u < u1) {
      Req r;
      load_req(a, req, r);
      const Shape s = shape_of(a, r);
      const int64_t units = s.units(weights);
      if (off >= units * a.KVH) {
        req++;
        off = 0;
        continue;
      }
      it.kvh = (int)div_pos(off, units);
      int64_t rest = off - it.kvh * units;
      int group = 0, tiles, w;
#pragma unroll 1
      for (;; group++) {
        tiles = group_tiles(a, r, s.rows, group);
        w = weights.of(s.rows, group);
        if (rest < (int64_t)tiles * w) break;
        rest -= (int64_t)tiles * w;
      }
      // the tiles whose first unit is in the share: an earlier share holds that of a tile cut at its start
      const int64_t base = u - rest;
      auto ceil_w = [&](int x) { return w == 1 ? x : w == 2 ? (x + 1) >> 1 : (x + 2) / 3; };
      const int t0 = ceil_w((int)rest), t1 = ceil_w((int)min(rest + (u1 - u), (int64_t)tiles * w));
      const int64_t step = min((int64_t)tiles * w - rest, u1 - u);
      u += step;
      off += step;
      if (t0 >= t1) continue;
      it.req = req;
      it.first = r.first;
      it.shift = r.len - r.n;
      it.len = r.len;
      it.row0 = group * 2 * kTcRows;
      it.rows = s.rows;
      it.t0 = t0;
      it.t1 = t1;
      it.whole = it.t0 == 0 && it.t1 == tiles;
      it.c0 = it.c1 = blockIdx.x;
      if (t0 > 0) it.c0 = (int)div_pos((base + 1) * G - 1, total);
      if (t1 < tiles) it.c1 = (int)div_pos((base + (int64_t)(tiles - 1) * w + 1) * G - 1, total);
      for (int t = 0; t < 2; t++) {
        const int row0 = it.row0 + t * kTcRows, last = min(s.rows, row0 + kTcRows) - 1;
        const int keys = it.shift + a.heads.div(last) + 1;  // that the tile's last row attends
        it.end[t] = row0 < s.rows ? max(it.t0, min(it.t1, (keys + kTcKeys - 1) / kTcKeys)) : it.t0;
      }
      it.split = it.row0 + kTcRows >= s.rows && it.end[0] - it.t0 >= 2;
      if (it.split) it.end[1] = it.end[0];
      stopped = false;
      break;
    }
    it.stop = stopped;
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(&sh.item_full[i % kItems]);
    return true;
  };
  ok = publish(0);
#pragma unroll 1
  for (int i = 0; ok && !sh.items[i % kItems].stop; i++) {
    if (!stopped) ok = publish(i + 1);
    if (ok) ok = load_item(a, sh, tiles, 1, sh.items[i % kItems], J, bad);
  }
  load_end(a, sh, 1, J, ok, bad);
}

// Issues the products of query tile `tile`; the whole warp runs this. The named barriers that the softmax warps wait at are
// met whatever fails, so `ok` only stops the work between them.
__device__ __forceinline__ void issue_role(const AttnArgs& a, TcShared& sh, uint8_t* tiles, uint32_t tmem, int tile) {
  constexpr uint32_t is = idesc_f16(kTcRows, kTcKeys, false), ip = idesc_f16(kTcRows, kTcDim, true);
  const int lane = threadIdx.x & 31;
  // the same in every lane, and known to be: else each product would be wrapped in a loop over the lanes' values
  auto uniform = [](uint32_t x) { return __shfl_sync(0xffffffffu, x, 0); };
  const uint32_t leader = lane == 0, k_tiles = smem_u32(tiles), v_tiles = k_tiles + kTcStages * kTile;
  const uint32_t cs = uniform(tmem + col_s(tile)), cpv = uniform(tmem + col_pv(tile)), cq = uniform(tmem + col_q(tile));
  bool ok = true;
  int J = 0, C = 0;
  auto wait_split = [&](int op, int j) {
    return warp_wait_bar(&sh.conv[op][j % kTcStages], (j / kTcStages) & 1, &sh.abort);
  };
  // the CTA's key tiles [j, end) that this query tile does not use: its share of freeing them, once they are split
  auto skip = [&](int j, int end) {
#pragma unroll 1
    for (; ok && j < end; j++)
#pragma unroll 1
      for (int op = 0; op < 2 && ok; op++) {
        ok = wait_split(op, j);
        if (ok && lane == 0) mbar_arrive(&sh.empty[op][j % kTcStages]);
      }
  };
  const Item* p_it;
  for (int i = 0; (p_it = take_item(sh, i)) != nullptr; free_item(sh, i), i++) {
    const Item it = *p_it;
    const int first = it.row0 + (it.split ? 0 : tile * kTcRows), next = J + it.t1 - it.t0;
    if (first >= it.rows) {
      skip(J, next);
      J = next;
      continue;
    }
    const int step = it.split ? 2 : 1, t0 = it.t0 + (it.split ? tile : 0);
    const int end = t0 + (max(0, (tile == 0 ? it.end[0] : it.end[1]) - t0) + step - 1) / step * step;
    const int threads = 64 * min(4, (it.rows - first + 31) >> 5) + 32;
    bar_named(kBarIssue + tile, threads);  // Q is in TMEM
#pragma unroll 1
    for (int t = t0; t < end; t += step, C++) {
      const int j = J + t - it.t0, st = j % kTcStages;
      if (t == t0) ok = ok && wait_split(0, j);
      ok = ok && (C == 0 || warp_wait_bar(&sh.pv_full[tile], (C - 1) & 1, &sh.abort));  // the last P has been read
      if (ok) {
        fence_after();
        const uint32_t kh = uniform(k_tiles + st * kTile);
#pragma unroll 1
        for (uint32_t i = 0; i < 3; i++) {  // lo·hi, hi·lo, hi·hi: the small ones first
          const uint32_t q = cq + (i == 0 ? 32u : 0u);
          const uint64_t k = desc_split(kh + (i == 1 ? kLo : 0u));
#pragma unroll
          for (uint32_t e = 0; e < 4; e++) mma_f16_ts(cs, q + 8 * e, k + 2 * e, is, i + e, leader);
        }
        commit_if(&sh.s_full[tile], leader);
        commit_if(&sh.empty[0][st], leader);
        if (it.split) commit_if(&sh.empty[0][st], leader);  // the other query tile's share as well
        ok = wait_split(1, j) && (t + step >= end || wait_split(0, j + step));  // here, where there is time
      }
      bar_named(kBarIssue + tile, threads);  // P is in TMEM
      if (ok) {
        fence_after();
        const uint32_t vh = uniform(v_tiles + st * kTile);
#pragma unroll 1
        for (uint32_t i = 0; i < 3; i++) {
          // 16 keys per product: columns 16 e of P's hi part, 8 further of its lo part
          const uint32_t w = cs + (i == 0 ? 8u : 0u);
          const uint64_t v = desc_split(vh + (i == 1 ? kLo : 0u));
#pragma unroll
          for (uint32_t e = 0; e < 8; e++) mma_f16_ts(cpv, w + 16 * e, v + (2 * kGroup >> 4) * e, ip, i + e, leader);
        }
        commit_if(&sh.pv_full[tile], leader);
        commit_if(&sh.empty[1][st], leader);
        if (it.split) commit_if(&sh.empty[1][st], leader);
      }
    }
    bar_named(kBarEnd + tile, 256 + 32);
    if (!it.split) skip(J + end - it.t0, next);
    J = next;
  }
  if (!ok && lane == 0) {
    atomicExch(a.error_flag, 79);
    sh.abort = 1;
  }
  // every product issued completes before the CTA gives its tensor memory back
  commit_if(&sh.drained[tile], leader);
  tc::warp_wait(&sh.drained[tile], 0);
}

__global__ void __launch_bounds__(kTcThreads, 1) k_paged_tc(const AttnArgs a) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  // an offset, not an address rounded up as an integer: the compiler then knows all of it for shared memory
  uint8_t* tiles = smem_raw + (-smem_u32(smem_raw) & 1023u);
  TcShared& sh = *reinterpret_cast<TcShared*>(tiles + 2 * kTcStages * kTile);
  const int tid = threadIdx.x, warp = tid >> 5;
  if (tid == 0) {
    for (int op = 0; op < 2; op++)
      for (int i = 0; i < kTcStages; i++) {
        mbar_init(&sh.raw[op][i], 1);
        mbar_init(&sh.conv[op][i], kConvWarps);
        mbar_init(&sh.empty[op][i], 2);
      }
    for (int i = 0; i < kItems; i++) {
      mbar_init(&sh.item_full[i], 1);
      mbar_init(&sh.item_free[i], kWalkWarp);  // every warp before the walking one takes each item
    }
    for (int t = 0; t < 2; t++) {
      mbar_init(&sh.s_full[t], 1);
      mbar_init(&sh.pv_full[t], 1);
      mbar_init(&sh.drained[t], 1);
    }
    sh.abort = 0;
    sh.unplaced = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) tc::tmem_alloc(&sh.tmem, 512);
  pdl_trigger();
  pdl_wait();
  __syncthreads();  // `unplaced` is set below

  // this CTA's share of the units
  const int per = (a.n + kTcThreads - 1) / kTcThreads;
  const int i0 = min(a.n, tid * per), i1 = min(a.n, i0 + per);
  int64_t count[2] = {0, 0}, count_before[2], all[2];  // key tiles of groups of one, of two query tiles
#pragma unroll 1
  for (int i = i0; i < i1; i++) {
    Req r;
    if (!load_req(a, i, r)) atomicExch(a.error_flag, 74);
    if (!r.placed) sh.unplaced = 1;
    const Shape s = shape_of(a, r);
    count[0] += s.ones * a.KVH;
    count[1] += s.twos * a.KVH;
  }
  block_prefix<kTcThreads>(count, sh.tmp, count_before, all);
  if (!sh.unplaced) zero_rest(a);
  const bool few = all[0] + all[1] <= 2 * (int64_t)gridDim.x;
  const Weights weights = few ? Weights{1, 1} : Weights{2, 3};
  const int64_t mine = count[0] * weights.one + count[1] * weights.two;
  const int64_t before = count_before[0] * weights.one + count_before[1] * weights.two;
  const int64_t total = all[0] * weights.one + all[1] * weights.two;
  // with two units or more per tile there are enough for each share to hold some tile's first unit
  const int64_t G = min((int64_t)gridDim.x, total), c = blockIdx.x;
  const int64_t u0 = div_pos(c * total, max(G, (int64_t)1)), u1 = div_pos((c + 1) * total, max(G, (int64_t)1));
  if (c < G && before <= u0 && u0 < before + mine) {
    int64_t off = u0 - before;
#pragma unroll 1
    for (int i = i0; i < i1; i++) {
      Req r;
      load_req(a, i, r);
      const int64_t units = shape_of(a, r).units(weights) * a.KVH;
      if (off < units) {
        sh.req = i;
        sh.off = off;
        break;
      }
      off -= units;
    }
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = sh.tmem;
  if (c < G) {
    if (warp < kConvWarp) {
      asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
      softmax_role(a, sh, tmem);
    } else if (warp < kLoadWarp) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kConvRegs));
      convert_role(a, sh, tiles, (warp - kConvWarp) / kConvWarps);
    } else {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kMiscRegs));
      if (warp == kLoadWarp) load_k_role(a, sh, tiles);
      else if (warp < kWalkWarp) issue_role(a, sh, tiles, tmem, warp - kIssueWarp);
      else walk_role(a, sh, tiles, sh.req, sh.off, u0, u1, total, G, weights);
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
