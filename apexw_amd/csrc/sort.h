// A stable sort of small integers by digits, for ids of experts and of words (gfx950).
//
// Items are given as ids; an id outside [0, limit) has the key `limit`, behind all others.  Each pass orders by one digit
// of up to 9 bits: a launch that counts each workgroup's digits and one that places its items.  There a workgroup adds up
// the counts of those before it by itself (64 workgroups' counts are 128 KB, read from L2), or, where more than kScan
// workgroups would each read that many, a launch in between does (8 M items of 64 experts 318 us without it, 82 with; at
// 800000 23 and 18, at 65536 the launch costs as much as it saves).  Up to 512 K items go in workgroups of 1024, more in
// workgroups of 4096 (262144 ids of 50000, two passes, 36 us by 1024, 47 by 4096; 800000 67 and 64).  The rank of an item
// among its wave's is counted from ballots of the digit's bits, so equal keys keep their order and equal calls give equal
// results.  Up to kSmall items go through all passes in one workgroup's LDS.
//
// What bounds it is the chain of launches and, in each, of dependent accesses: 16384 ids in two passes take 18 us, the
// counts' launches 3 to 4 and the places' 5.5 each, for 0.5 MB that they move.
#pragma once

#include "common.h"

namespace {

constexpr int kDigits = 512, kSortThreads = 512, kSortWaves = kSortThreads / 64;
constexpr int kFew = 2, kMost = 8;               // items of a thread
constexpr int kSmall = kSortThreads * kMost;     // items of one workgroup
constexpr int kScan = 64;

struct SortArgs {
  const void* ids;        // int32 or int64
  int32_t wide;           // int64
  int32_t n;
  uint32_t limit;
  int32_t bits, passes;   // of a digit
  u32x2* from;            // (key, item) of a pass after the first
  u32x2* to;
  uint32_t* counts;       // [workgroup][digit]; where there are more than kScan: of those before, and of all behind them
  char* clear;            // cleared on the way, an even number of bytes
  int64_t clears;
  int32_t *source, *place, *ends;   // of the last pass for experts
};

APEXW_DEV u32x2 sort_item(const SortArgs& a, int i) {
  uint32_t key;
  if (a.wide) {
    const int64_t id = APEXW_GLOBAL(const int64_t, a.ids)[i];
    key = (uint64_t)id < a.limit ? (uint32_t)id : a.limit;
  } else {
    const uint32_t id = APEXW_GLOBAL(const uint32_t, a.ids)[i];
    key = id < a.limit ? id : a.limit;
  }
  return u32x2{key, (uint32_t)i};
}

// lanes of the wave whose digit is this lane's, of those that `valid` names
APEXW_DEV uint64_t same_digit(uint32_t d, int bits, uint64_t valid) {
  uint64_t mask = valid;
  for (int b = 0; b < bits; ++b) {
    const uint64_t set = __ballot(d >> b & 1u);
    mask &= d >> b & 1u ? set : ~set;
  }
  return mask;
}

// Exclusive prefix sum over the workgroup's threads; lds: one value a wave.  All threads call it.
APEXW_DEV uint32_t sort_scan(uint32_t x, uint32_t* lds) {
  uint32_t up = x;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint32_t y = __shfl_up(up, off, 64);
    if (lane_id() >= off) up += y;
  }
  const int wave = threadIdx.x >> 6;
  if (lane_id() == 63) lds[wave] = up;
  __syncthreads();
  uint32_t before = 0;
  for (int w = 0; w < wave; ++w) before += lds[w];
  __syncthreads();
  return before + up - x;
}

struct SortLds {
  uint32_t cnt[kSortWaves][kDigits];
  uint32_t wave[kSortWaves];
};

// One pass over the items of this workgroup: rounds x 64 consecutive ones a wave from `first` on, get(i) the item i.
// put(item, position, start of its digit's block) places each.  kAlone: the workgroup has all items.
// digit_end(d, end): thread d gets the end of digit d's block.
template <bool kAlone, int kItems, class Get, class Put, class End>
APEXW_DEV void sort_pass(const SortArgs& a, SortLds& l, int pass, int first, int rounds, Get&& get, Put&& put,
                         End&& digit_end) {
  const int digits = 1 << a.bits, wave = threadIdx.x >> 6, lane = lane_id(), shift = pass * a.bits;
  const uint32_t low = (uint32_t)digits - 1u;
  for (int i = threadIdx.x; i < kSortWaves * digits; i += kSortThreads) l.cnt[i >> a.bits][i & low] = 0u;
  __syncthreads();
  u32x2 item[kItems];
  uint32_t rank[kItems];
  const int base = first + wave * rounds * 64 + lane;
#pragma unroll
  for (int r = 0; r < kItems; ++r)
    if (r < rounds && base + r * 64 < a.n) item[r] = get(base + r * 64);
#pragma unroll
  for (int r = 0; r < kItems; ++r) {
    if (r >= rounds) break;
    const bool valid = base + r * 64 < a.n;
    const uint32_t d = valid ? item[r][0] >> shift & low : 0u;
    const uint64_t mask = same_digit(d, a.bits, __ballot(valid));
    const uint32_t ahead = __builtin_popcountll(mask & ((1ull << lane) - 1ull));
    const uint32_t old = l.cnt[wave][d];
    rank[r] = old + ahead;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (valid && ahead == 0u) l.cnt[wave][d] = old + (uint32_t)__builtin_popcountll(mask);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
  __syncthreads();
  // thread d: the digit's items in the waves before, in the workgroups before, and in all
  const int d = threadIdx.x;
  uint32_t mine = 0u, before = 0u, all = 0u;
  if (d < digits) {
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) {
      const uint32_t c = l.cnt[w][d];
      l.cnt[w][d] = mine;
      mine += c;
    }
    if (kAlone) {
      all = mine;
    } else if (gridDim.x > kScan) {
      before = a.counts[(int64_t)blockIdx.x * digits + d], all = a.counts[(int64_t)gridDim.x * digits + d];
    } else {
      constexpr int U = 16;   // loads in flight
      for (int b0 = 0; b0 < (int)gridDim.x; b0 += U) {
        uint32_t c[U];
#pragma unroll
        for (int u = 0; u < U; ++u) c[u] = b0 + u < (int)gridDim.x ? a.counts[(int64_t)(b0 + u) * digits + d] : 0u;
#pragma unroll
        for (int u = 0; u < U; ++u) all += c[u], before += b0 + u < (int)blockIdx.x ? c[u] : 0u;
      }
    }
  }
  const uint32_t start = sort_scan(all, l.wave);
  if (d < digits) {
    digit_end(d, start + all);
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) l.cnt[w][d] += start + before;
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kItems; ++r)
    if (r < rounds && base + r * 64 < a.n) put(item[r], l.cnt[wave][item[r][0] >> shift & low] + rank[r]);
}

// kClear bytes in a row at a time (the last chunk overlaps the one before).  1 GB: 16 KB 175 us, 8 204, 32 188, 64 190.
constexpr int64_t kClear = 2 * kSortThreads * 16;
APEXW_DEV void sort_clear(const SortArgs& a, int64_t group, int64_t groups) {
  struct __attribute__((packed, aligned(2))) Chunk2 { u32x4 v; };
  const int64_t last = a.clears - 16;
  for (int64_t from = group * kClear; from < a.clears; from += groups * kClear)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t at = from + (i * kSortThreads + threadIdx.x) * 16;
      if (at >= a.clears) break;
      if (last >= 0) APEXW_GLOBAL(Chunk2, a.clear + (at < last ? at : last))->v = u32x4{0u, 0u, 0u, 0u};
      else for (int64_t j = 0; j < a.clears; j += 2) *APEXW_GLOBAL(uint16_t, a.clear + j) = 0;
    }
}

// The counts of each workgroup's digits
template <bool kFirst, int kItems> __global__ __launch_bounds__(kSortThreads) void sort_count_kernel(SortArgs a, int pass) {
  __shared__ uint32_t cnt[kDigits];
  const int digits = 1 << a.bits, shift = pass * a.bits, first = blockIdx.x * kSortThreads * kItems;
  if (kFirst) sort_clear(a, blockIdx.x, gridDim.x);
  for (int i = threadIdx.x; i < digits; i += kSortThreads) cnt[i] = 0u;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kItems; ++r) {
    const int i = first + r * kSortThreads + threadIdx.x;
    if (i >= a.n) continue;
    const uint32_t key = kFirst ? sort_item(a, i)[0] : a.from[i][0];
    atomicAdd(&cnt[key >> shift & (uint32_t)(digits - 1)], 1u);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < digits; i += kSortThreads) a.counts[(int64_t)blockIdx.x * digits + i] = cnt[i];
}

// The counts of many workgroups added up: a lane has a digit, a wave a 16th of the workgroups
__global__ __launch_bounds__(1024) void sort_scan_kernel(uint32_t* counts, int groups, int digits) {
  __shared__ uint32_t sums[16][64];
  const int wave = threadIdx.x >> 6, lane = lane_id(), d = blockIdx.x * 64 + lane;
  const int len = (groups + 15) / 16, g0 = wave * len, g1 = g0 + len < groups ? g0 + len : groups;
  constexpr int U = 16;   // loads in flight
  uint32_t* at = counts + d;
  uint32_t sum = 0u;
  if (d < digits)
    for (int g = g0; g < g1; g += U) {
      uint32_t c[U];
#pragma unroll
      for (int u = 0; u < U; ++u) c[u] = g + u < g1 ? at[(int64_t)(g + u) * digits] : 0u;
#pragma unroll
      for (int u = 0; u < U; ++u) sum += c[u];
    }
  sums[wave][lane] = sum;
  __syncthreads();
  if (d >= digits) return;
  uint32_t before = 0u;
  for (int w = 0; w < wave; ++w) before += sums[w][lane];
  if (wave == 15) at[(int64_t)groups * digits] = before + sum;
  for (int g = g0; g < g1; g += U) {
    uint32_t c[U];
#pragma unroll
    for (int u = 0; u < U; ++u) c[u] = g + u < g1 ? at[(int64_t)(g + u) * digits] : 0u;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (g + u < g1) at[(int64_t)(g + u) * digits] = before, before += c[u];
  }
}

// where the last pass puts an item for experts
APEXW_DEV void sort_order(const SortArgs& a, u32x2 item, uint32_t at) {
  const bool none = item[0] == a.limit;
  APEXW_GLOBAL(int32_t, a.source)[at] = none ? -1 : (int32_t)item[1];
  APEXW_GLOBAL(int32_t, a.place)[item[1]] = none ? -1 : (int32_t)at;
}

// kOrder: the last pass of an experts' order, whose ends are the digits' where one pass sorts them
template <bool kFirst, bool kOrder, int kItems> __global__ __launch_bounds__(kSortThreads) void sort_place_kernel(SortArgs a, int pass) {
  __shared__ SortLds l;
  sort_pass<false, kItems>(
      a, l, pass, blockIdx.x * kSortThreads * kItems, kItems, [&](int i) { return kFirst ? sort_item(a, i) : a.from[i]; },
      [&](u32x2 item, uint32_t at) {
        if (kOrder) sort_order(a, item, at);
        if (a.to) a.to[at] = item;
      },
      [&](int d, uint32_t end) {
        if (kOrder && a.passes == 1 && blockIdx.x == 0 && (uint32_t)d < a.limit) a.ends[d] = (int32_t)end;
      });
}

// All passes of up to kItems items a thread in one workgroup
template <bool kOrder, int kItems> APEXW_DEV void sort_small(const SortArgs& a) {
  __shared__ SortLds l;
  __shared__ u32x2 items[kItems * kSortThreads];
  const int rounds = (a.n + kSortThreads - 1) / kSortThreads;
  for (int pass = 0; pass < a.passes; ++pass) {
    const bool last = pass == a.passes - 1;
    sort_pass<true, kItems>(
        a, l, pass, 0, rounds, [&](int i) { return pass == 0 ? sort_item(a, i) : items[i]; },
        [&](u32x2 item, uint32_t at) {
          if (!last) items[at] = item;
          else if (kOrder) sort_order(a, item, at);
          if (last && a.to) a.to[at] = item;
        },
        [&](int d, uint32_t end) {
          if (kOrder && a.passes == 1 && (uint32_t)d < a.limit) a.ends[d] = (int32_t)end;
        });
    __syncthreads();
  }
}

inline void sort_digits(SortArgs& a) {
  int bits = 1;
  while (bits < 32 && (uint64_t)a.limit >> bits) ++bits;   // of the keys 0 .. limit
  a.passes = (bits + 8) / 9;
  a.bits = (bits + a.passes - 1) / a.passes;
}
// items of a thread, workgroups of a pass
inline int sort_items(int64_t n) { return n <= 512 * kSortThreads * kFew ? kFew : kMost; }
inline int sort_groups(int64_t n) {
  const int64_t per = kSortThreads * sort_items(n);
  return (int)((n + per - 1) / per);
}

}  // namespace
