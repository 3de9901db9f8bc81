// Tiles of matrix products grouped by expert, one group or many (gfx950): which tiles a workgroup has, the stream of
// asynchronous copies, LDS reads and matrix instructions that computes them, and how a product is cut.
//
// The kernels that use it say where a tile's operands lie (`locate`) and what becomes of it (`out`).
#pragma once

#include <cmath>
#include <type_traits>

#include "common.h"

int apexw_cu_count();

namespace {

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(4))) short v4i16;

struct ExpertArgs {
  const uint16_t *a, *b;      // rows product: rows and weights; weight grad: dy and x
  const int32_t* ends;
  void* out;
  int64_t lda, ldb, sb, ldo;  // row strides; expert stride of the weights
  int64_t rows;
  int32_t experts, n, k;      // out [rows x n] over k, or [experts x n x k]
  int32_t wide;               // k, or the k that rows copied for their alignment were filled up to with zeros
  // a product whose tiles are few is cut along what it sums over: `splits` parts (of `part` k in a rows product,
  // of an expert's rows in a weight grad) leave fp32 sums split_stride elements apart, which join_* add up
  int32_t splits, part;
  int64_t split_stride;
  int32_t which;              // kAll, or the two launches that kMost and kRest make of a rows product's tiles
};

// Tiles of 256 rows take nearly the same time however few rows they hold (a stage waits for its copies), so a
// launch of them leaves last tiles of up to 128 rows to a second launch, of 128-row tiles.
constexpr int kAll = 0, kMost = 1, kRest = 2;

APEXW_DEV int wave_prefix_max(int x) {
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int y = __shfl_up(x, off, 64);
    if (lane_id() >= off && y > x) x = y;
  }
  return x;
}
APEXW_DEV int wave_prefix_sum(int x) {
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int y = __shfl_up(x, off, 64);
    if (lane_id() >= off) x += y;
  }
  return x;
}
APEXW_DEV int lane_of(int x, int l) { return __builtin_amdgcn_readlane(x, l); }

// The rows [begin, end) of 64 experts from e0 on, a lane each (behind the last one: no rows); row: the end of
// the ones before, then of these
APEXW_DEV void look(const ExpertArgs& g, int e0, int& row, int& begin, int& end) {
  const int e = e0 + lane_id(), most = (int)g.rows;
  end = e < g.experts ? g.ends[e] : row;
  end = wave_prefix_max(end > most ? most : end < row ? row : end);
  begin = __shfl_up(end, 1, 64);
  if (lane_id() == 0) begin = row;
  row = lane_of(end, 63);
}

struct Job {
  int expert;          // -1: none
  int first, last;     // its rows
  int row, col;        // the tile's first row among its rows; its place across, in tiles
  int split;           // which part of what is summed over
};

// Tile (row, column) of index t among rows x cols tiles: bands of 8 tile rows, column by column, so that the
// tiles that run at a time share both operands' lines in L2
APEXW_DEV void place(int t, int rows, int cols, int& r, int& c) {
  const int band = t / (8 * cols), in = t - band * 8 * cols;
  const int high = rows - band * 8 < 8 ? rows - band * 8 : 8;
  c = in / high;
  r = band * 8 + in - c * high;
}

// The tiles of a rows product, expert by expert.  Workgroups go to the 8 XCDs in turn: each XCD gets a
// contiguous part of the tiles, of which its workgroups take every (number of them)th.
template <bool kCut> struct RowJobs {
  const ExpertArgs& g;
  int size, cols;              // rows of a tile, tiles across
  int begin, end, upto;        // per lane, of the first 64 experts: rows, and tiles up to and with it
  int all, rows;               // tiles, and rows that belong to experts

  __device__ __forceinline__ RowJobs(const ExpertArgs& a, int bm, int bn)
      : g(a), size(bm), cols((a.n + bn - 1) / bn), all(0), rows(0) {
    for (int e0 = 0; e0 < g.experts; e0 += 64) step(e0);
  }
  // tile rows of n rows of an expert
  __device__ __forceinline__ int high(int n) const {
    if (g.which == kMost) return n / 256 + (n % 256 > 128);
    if (g.which == kRest) return n % 256 > 0 && n % 256 <= 128;
    return (n + size - 1) / size;
  }
  __device__ __forceinline__ void step(int e0) {
    look(g, e0, rows, begin, end);
    upto = all + wave_prefix_sum(high(end - begin) * cols);
    all = lane_of(upto, 63);
  }
  __device__ __forceinline__ int find_at(int t, int e0, Job& j) const {
    const uint64_t hit = __ballot(t < upto);
    if (!hit) return 0;
    const int l = __builtin_ctzll(hit);
    j.expert = e0 + l, j.first = lane_of(begin, l), j.last = lane_of(end, l);
    const int down = high(j.last - j.first);
    place(t - (lane_of(upto, l) - down * cols), down, cols, j.row, j.col);
    j.row = g.which == kRest ? (j.last - j.first) / 256 * 256 : j.row * size;
    return 1;
  }
  // the i-th tile of this workgroup.  Round i's tiles go to the XCD's workgroups in turn from another one on
  // each time, since a tile of few rows takes less time and stands at the same place of every column; where
  // the last round has tiles for less than half or a quarter of them, it takes halves or quarters of tiles.
  __device__ __forceinline__ Job get(int i) {
    Job j{-1, 0, 0, 0, 0, 0};
    const int units = all * g.splits, part = (units + 7) / 8, from = (int)(blockIdx.x % 8) * part;
    const int groups = (int)(gridDim.x / 8), mine = units - from < part ? units - from : part;
    int in = i * groups + (int)((blockIdx.x / 8 + 5u * i) % groups), sub = 0, cut = 1;
    const int rest = mine - i * groups;
    if (kCut && g.splits == 1 && rest > 0 && 2 * rest <= groups) {
      cut = 4 * rest <= groups ? 4 : 2;
      sub = (in - i * groups) % cut, in = i * groups + (in - i * groups) / cut;
    }
    if (in >= mine) return j;
    const int t = (from + in) / g.splits;
    j.split = (from + in) % g.splits;
    if (g.experts <= 64) {
      find_at(t, 0, j);
    } else {
      const int keep_all = all, keep_rows = rows;
      all = rows = 0;
      for (int e0 = 0; e0 < g.experts; e0 += 64) {
        step(e0);
        if (find_at(t, e0, j)) break;
      }
      all = keep_all, rows = keep_rows;
    }
    if (cut > 1) {
      const int end = j.first + j.row + (sub + 1) * (size / cut);
      j.row += sub * (size / cut);
      j.last = j.last < end ? j.last : end;
      if (j.first + j.row >= j.last) j.last = j.first;   // no rows in this part: nothing to do
    }
    return j;
  }
};

// the rows of a part of an expert's: whole stages
APEXW_DEV int split_rows(int rows, int splits) { return ((rows + splits - 1) / splits + 63) / 64 * 64; }

// The tiles of a weight gradient.  Experts differ in rows, and so their tiles in work: each XCD takes a part of
// every expert's tiles, and up to 64 experts come in the order of their rows, the most first, so that the
// last tiles are short.  Experts of few tiles would leave XCDs without any (32 of 256 x 256, two tiles each,
// 16384 rows: 46 us), so those are dealt out one by one (17 us).
struct WeightJobs {
  const ExpertArgs& g;
  int size, high, cols, part;
  int begin, end, rank;        // per lane, of the first 64 experts
  int next_rank;               // experts that have rows

  __device__ __forceinline__ WeightJobs(const ExpertArgs& a, int bm, int bn)
      : g(a), size(bm), high((a.n + bm - 1) / bm), cols((a.k + bn - 1) / bn) {
    part = (high * cols * g.splits + 7) / 8;
    int row = 0;
    look(g, 0, row, begin, end);
    rank = 0;
    for (int l = 0; l < 64; ++l) {
      const int n = lane_of(end - begin, l);
      rank += n > end - begin || (n == end - begin && l < lane_id());
    }
    next_rank = __builtin_popcountll(__ballot(end > begin));
  }
  __device__ __forceinline__ Job get(int i) const {
    Job j{-1, 0, 0, 0, 0, 0};
    // forth and back, so that the first workgroups do not get the most rows in every round
    const int groups = (int)(gridDim.x / 8), w = (int)(blockIdx.x / 8), in = i * groups + (i & 1 ? groups - 1 - w : w);
    const int units = high * cols * g.splits, x = (int)(blockIdx.x % 8);
    int t = x * part + in % part, e = in / part;
    if (units < 64) e = (8 * in + x) / units, t = (8 * in + x) % units;
    if (g.experts <= 64) {
      if (e >= next_rank) return j;
      e = __builtin_ctzll(__ballot(rank == e));
      j.first = lane_of(begin, e), j.last = lane_of(end, e);
    } else {
      if (e >= g.experts) return j;
      int row = 0, b, n;
      for (int e0 = 0; e0 <= e; e0 += 64) look(g, e0, row, b, n);
      j.first = lane_of(b, e & 63), j.last = lane_of(n, e & 63);
    }
    j.expert = e;
    if (t >= units) {
      j.last = j.first;   // no tile here: nothing to do
      return j;
    }
    place(t / g.splits, high, cols, j.row, j.col);
    j.row *= size;
    if (g.splits > 1) {
      j.split = t % g.splits;
      const int len = split_rows(j.last - j.first, g.splits), from = j.split * len, n = j.last - j.first - from;
      j.first += from < j.last - j.first ? from : j.last - j.first;
      j.last = j.first + (n <= 0 ? 0 : n < len ? n : len);
    }
    return j;
  }
};

struct __attribute__((packed, aligned(2))) Chunk { u32x4 v; };
struct __attribute__((packed, aligned(4))) Chunk32 { u32x4 v; };

// 8 elements from p, those below cnt (the rest 0), at any element address
APEXW_DEV u32x4 load_chunk(const uint16_t* p, int cnt) {
  if (cnt >= 8) return APEXW_GLOBAL(const Chunk, p)->v;
  u32x4 r = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < cnt) r[j >> 1] |= (uint32_t)APEXW_GLOBAL(const uint16_t, p)[j] << (16 * (j & 1));
  return r;
}

APEXW_DEV int clamp8(int64_t left) { return left <= 0 ? 0 : left < 8 ? (int)left : 8; }

template <int DT> APEXW_DEV f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (DT == APEXW_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

template <int OD> APEXW_DEV void store_elem(void* base, int64_t i, float x) {
  if constexpr (OD == APEXW_F32) APEXW_GLOBAL(float, base)[i] = x;
  else if constexpr (OD == APEXW_BF16) APEXW_GLOBAL(uint16_t, base)[i] = (uint16_t)f32_to_bf16_bits(x);
  else APEXW_GLOBAL(uint16_t, base)[i] = (uint16_t)f32_to_f16_bits(x);
}

// ---------------------------------------------------------------------------
// Aligned operands: tiles of BM x BN staged by asynchronous copies
// ---------------------------------------------------------------------------

// 16 bytes a lane from a buffer to LDS: lane L's at byte voff past the buffer's base land at LDS byte
// lds_base + 16 L, zeros where voff is past the buffer's end.  In assembly so that the compiler does not make
// every later LDS read wait for it; the kernel orders the copies itself (a stage is read after the wait and
// the barrier that follow its copies, and refilled after the barrier that follows its last reads).
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
APEXW_DEV void lds_copy16(uint32_t lds_base, uint32_t voff, u32x4 buffer) {
  lds_base = uniform(lds_base);
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :
               : "s"(lds_base), "v"(voff), "s"(buffer)
               : "memory", "m0");
}
#pragma clang diagnostic pop

template <int N> APEXW_DEV void wait_copies() {
  static_assert(N >= 0 && N < 64, "vmcnt");
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// lgkmcnt(0) by the builtin, so that the compiler knows that this wave's LDS reads are back
APEXW_DEV void barrier() {
  __builtin_amdgcn_s_waitcnt(0xC07F);
  asm volatile("s_barrier" ::: "memory");
}

constexpr int kDepth = 64;              // k of a stage: a row's 128 bytes, one cache line
constexpr uint32_t kNowhere = 0xFFFFFFF0u;   // a buffer offset past every end

APEXW_DEV uint64_t uniform64(uint64_t x) { return (uint64_t)uniform((uint32_t)(x >> 32)) << 32 | uniform((uint32_t)x); }

// The memory of one operand of a tile: its origin (row or column 0, k 0), the bytes from there to its end, its
// stages and the k of the last one
struct Span {
  const uint16_t* base;
  int64_t left;
  int stages, tail;
  __device__ __forceinline__ void fix() {   // into scalar registers
    base = (const uint16_t*)uniform64((uint64_t)base), left = (int64_t)uniform64((uint64_t)left);
    stages = uniform(stages), tail = uniform(tail);
  }
  // rows: rows (columns) from the origin on; depth: k; ld: elements from row to row (k row to k row).  What a stage
  // brings of k rows behind the last one is left out by the end of the memory alone: k rows may not overlap.
  template <bool kKN> __device__ __forceinline__ void set(const uint16_t* p, int64_t ld, int64_t rows, int depth, int size) {
    base = p;
    left = kKN ? ((depth - 1) * ld + rows) * 2 : (((rows < size ? rows : size) - 1) * ld + depth) * 2;
    stages = (depth + kDepth - 1) / kDepth;
    tail = (depth - 1) % kDepth + 1;
  }
};

// How one operand of a tile gets into LDS and out: kSize of its rows (or, kKN, columns) over the k of a stage.
//   k-contiguous: LDS [kSize rows][64 k]; the 8 chunks of row r are swapped by XOR with (r / 2) % 8, so that the
//     fragment reads of 16 consecutive rows touch every bank once
//   kKN: LDS [64 k][kSize columns]; the chunks of k row r are swapped by XOR with 4 (r % 4) + 2 (r / 8 % 2), so
//     that the transposing reads of rows r .. r + 3 and r + 8 .. r + 11 do
template <bool kKN, int kSize, int kWaves> struct Operand {
  static constexpr int kElems = kSize * kDepth;            // of a stage
  static constexpr int kCopies = kSize / 8 / kWaves;       // of a wave and stage, 1 KB each
  int64_t step;           // bytes from stage to stage
  uint32_t voff[kCopies]; // per lane
  uint32_t lds0;          // of this wave's first copy in stage 0

  __device__ __forceinline__ void init(int64_t ld, const uint16_t* lds) {
    const int lane = lane_id(), wave = threadIdx.x >> 6;
    step = (kKN ? (int64_t)kDepth * ld : kDepth) * 2;
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
      const int q = wave * kCopies + i;
      if constexpr (kKN) {
        constexpr int kChunks = kSize / 8;
        const int k = q * (64 / kChunks) + lane / kChunks, chunk = (lane % kChunks) ^ swap(k);
        voff[i] = (uint32_t)(k * ld + chunk * 8) * 2u;
      } else {
        voff[i] = (uint32_t)((q * 8 + (lane >> 3)) * ld + chunk_of(i) * 8) * 2u;
      }
    }
    lds0 = uniform((uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)(lds + wave * kCopies * 512));
  }
  __device__ __forceinline__ int chunk_of(int i) const {   // k-contiguous: the chunk that this lane's copy i brings
    const int lane = lane_id(), q = (threadIdx.x >> 6) * kCopies + i;
    return (lane & 7) ^ ((4 * (q & 1) + (lane >> 4)) & 7);
  }
  __device__ __forceinline__ u32x4 buffer(const Span& m, int h) const {
    const uint64_t at = (uint64_t)m.base + (uint64_t)(h * step);
    int64_t n = m.left - h * step;
    n = n < 0 ? 0 : n > 0xFFFFFF00ll ? 0xFFFFFF00ll : n;
    return u32x4{uniform((uint32_t)at), uniform((uint32_t)(at >> 32)), uniform((uint32_t)n), 0x00020000u};
  }
  // copy i of a stage into the buffer at LDS byte `to`; tail: the k that exist in this stage
  __device__ __forceinline__ void copy(u32x4 b, int i, uint32_t to, int tail) const {
    uint32_t v = voff[i];
    if constexpr (!kKN) v = chunk_of(i) * 8 >= tail ? kNowhere : v;
    lds_copy16(lds0 + to + i * 1024, v, b);
  }
  static __device__ __forceinline__ int swap(int k) { return 4 * (k & 3) + 2 * (k >> 3 & 1); }
  // the fragment of 16 rows (columns) from `row` at step s of 32 k: lane l has row l % 16, k = 8 (l / 16) .. + 7.
  // From [k][column] by two transposing reads: in each 16 lanes, lane 4 r + c gets element c of the 8-byte rows
  // that lanes r, r + 4, r + 8, r + 12 address.
  static __device__ __forceinline__ u32x4 frag(const uint16_t* lds, int row, int s) {
    const int lane = lane_id();
    if constexpr (kKN) {
      const int r = lane & 3, k = 32 * s + 8 * (lane >> 4) + (lane >> 2 & 3), n = row + 4 * r;
      const int e = k * kSize + (((n >> 3) ^ swap(k)) << 3) + (n & 7);
      const v4i16 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4i16*)&lds[e]);
      const v4i16 hi =
          __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4i16*)&lds[e + 4 * kSize]);
      const u32x2 wl = __builtin_bit_cast(u32x2, lo), wh = __builtin_bit_cast(u32x2, hi);
      return u32x4{wl[0], wl[1], wh[0], wh[1]};
    } else {
      const int r = row + (lane & 15), c = (4 * s + (lane >> 4)) ^ ((lane >> 1) & 7);   // row: a multiple of 16
      return *(const u32x4*)&lds[r * kDepth + c * 8];
    }
  }
};

// A tile's shape: BM x BN by waves of WM x WN; LDS holds kStages stages of 64 k and 16 rows of 128 bytes of each
// wave's output
template <int BM_, int BN_, int WM_, int WN_, int kStages_, int kPerCU_> struct Shape {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, kStages = kStages_, kPerCU = kPerCU_;
  static constexpr int kWaves = (BM / WM) * (BN / WN), kThreads = kWaves * 64;
  static constexpr int kStageElems = (BM + BN) * kDepth, kOut = 16 * 64, kLds = kStages * kStageElems + kWaves * kOut;
  static_assert(kLds * 2 * kPerCU <= 160 * 1024, "LDS of a CU");
};
typedef Shape<256, 256, 128, 64, 2, 1> Large;
typedef Shape<128, 256, 64, 64, 3, 1> Wide;
typedef Shape<64, 128, 32, 64, 3, 2> Mid;
typedef Shape<32, 128, 32, 32, 3, 2> Small;

// What becomes of a tile.  A policy's Rows are what it loads of the rows of its lane's blocks when the tile begins;
// stores() says how many stores a wave makes of a whole tile.  Here: the tile as it is, or what `value` makes of the four
// sums of a lane, added to what is there (kAdd, fp32), in whole lines.  value(v, r, c): columns c .. c + 3 of the tile's
// row r.
struct Same {
  __device__ __forceinline__ f32x4 operator()(f32x4 v, int, int) const { return v; }
};
struct NoRows {   // nothing is known of a tile's rows beforehand
  __device__ __forceinline__ void arrived() const {}
};
template <int OD, bool kAdd = false> struct Store {
  template <int FA> using Rows = NoRows;
  template <class R> __device__ __forceinline__ void load(R&, int64_t, int, int) const {}
  template <class S> static constexpr int stores() { return S::WM / 16 * (S::WN * (OD == APEXW_F32 ? 4 : 2) / 64); }
  template <class S, int kWM, class Acc>
  __device__ __forceinline__ void write(const ExpertArgs& g, Acc& acc, const NoRows&, uint16_t* lds, int down, int across,
                                        int rows, int cols, int64_t out0) const {
    put<S, kWM>(g, acc, lds, down, across, rows, cols, out0, Same{});
  }

  // Lane l has row l % 16, columns 4 (l / 16) .. + 3 of a block.  Each wave puts 16 rows of 128 bytes into LDS of
  // its own, chunks swapped by XOR with the row, and writes them out in whole lines.
  // (Addresses are formed here, not kept in registers over the stages.)
  template <class S, int kWM, class Acc, class Value>
  static __device__ __forceinline__ void put(const ExpertArgs& g, const Acc& acc, uint16_t* lds, int down, int across,
                                             int rows, int cols, int64_t out0, Value&& value) {
    constexpr int FA = kWM / 16, FB = S::WN / 16;
    const int wm = down * kWM, wn = across * S::WN;
    uint16_t* mine = lds + S::kStages * S::kStageElems + (down * (S::BN / S::WN) + across) * S::kOut;
    int lane = lane_id();
    asm volatile("" : "+v"(lane));
    constexpr int kBlocks = OD == APEXW_F32 ? 2 : FB < 4 ? FB : 4, kPer = OD == APEXW_F32 ? 4 : 8;
    constexpr int kChunks = kBlocks * 16 / kPer, kRows = 64 / kChunks;   // of a staged row; rows of a store
    const int r0 = lane & 15, c0 = lane >> 4;
#pragma unroll
    for (int i = 0; i < FA; ++i)
#pragma unroll
      for (int j0 = 0; j0 < FB; j0 += kBlocks) {
#pragma unroll
        for (int j = 0; j < kBlocks; ++j) {
          const f32x4 v = value(acc[i][j0 + j], wm + 16 * i + r0, wn + 16 * (j0 + j) + 4 * c0);
          if constexpr (OD == APEXW_F32) {
            *(u32x4*)&mine[(r0 * kChunks + ((4 * j + c0) ^ (r0 & (kChunks - 1)))) * 8] =
                u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
          } else {
            u32x2 w;
            if constexpr (OD == APEXW_BF16) w = u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
            else
              w = u32x2{f32_to_f16_bits(v[0]) | (f32_to_f16_bits(v[1]) << 16),
                        f32_to_f16_bits(v[2]) | (f32_to_f16_bits(v[3]) << 16)};
            *(u32x2*)&mine[(r0 * kChunks + ((2 * j + (c0 >> 1)) ^ (r0 & (kChunks - 1)))) * 8 + 4 * (c0 & 1)] = w;
          }
        }
#pragma unroll
        for (int t = 0; t < 16 / kRows; ++t) {
          const int r = kRows * t + lane / kChunks, c = lane % kChunks;
          u32x4 w = *(const u32x4*)&mine[(r * kChunks + (c ^ (r & (kChunks - 1)))) * 8];
          const int row = wm + 16 * i + r, col = wn + 16 * j0 + kPer * c;
          if (row >= rows || col >= cols) continue;
          const int64_t o = out0 + row * g.ldo + col;
          if (col + kPer <= cols) {   // at any element address: rows of odd width start anywhere
            if constexpr (OD == APEXW_F32) {
              if constexpr (kAdd) {
                const u32x4 old = APEXW_GLOBAL(Chunk32, (float*)g.out + o)->v;
#pragma unroll
                for (int x = 0; x < 4; ++x) w[x] = __float_as_uint(__uint_as_float(old[x]) + __uint_as_float(w[x]));
              }
              APEXW_GLOBAL(Chunk32, (float*)g.out + o)->v = w;
            } else {
              APEXW_GLOBAL(Chunk, (uint16_t*)g.out + o)->v = w;
            }
          } else {
#pragma unroll
            for (int x = 0; x < kPer; ++x)
              if (col + x < cols) {
                if constexpr (OD == APEXW_F32) {
                  auto* p = APEXW_GLOBAL(uint32_t, g.out) + o + x;
                  *p = kAdd ? __float_as_uint(__uint_as_float(*p) + __uint_as_float(w[x])) : w[x];
                } else {
                  APEXW_GLOBAL(uint16_t, g.out)[o + x] = (uint16_t)(w[x >> 1] >> (16 * (x & 1)));
                }
              }
          }
        }
      }
  }
};

// The tiles of a workgroup, each A B^T over its k, as one stream of stages: the copies of a tile's first
// stages are under way while the tile before is multiplied and written out.
//
// A stage is two steps of 32 k by 16 x 16 x 32 MFMAs (at the power limit, which bounds large products of real
// numbers, they reach 2160 TFLOP/s from registers where 32 x 32 x 16 ones reach 1950).  After an MFMA come at
// most two fragment reads of the next step and one copy, fenced in place: issued in bursts they stall the
// wave's in-order issue.  The second step's fragments are in registers when it begins, so the barrier stands
// after its first two rows of products, where a wave has four of them and more (standing before them, the wait for
// the last reads and for the other waves found the matrix cores idle).  Behind it the stage's buffer is free for the
// copies of the stage kStages on, and the next stage, landed, gives its first fragments.  A's fragments are read into the
// registers of the ones just used.  Behind the last tile's stages come copies of no memory, which leave zeros: a test around each copy
// cost as much.
//
// Tried for 256 x 256 and not taken: a third stage of one operand, which leaves the copies two stages' time, with the
// tile written from registers (1% slower: their latency does not bound a stage); four waves of 128 x 128, whose
// fragments take two thirds of the LDS reads (the sums do not stay in place in 256 accumulation registers).
template <class S, bool kAKN, bool kBKN, int DT, bool kHalves, class Jobs, class Place, class Out>
APEXW_DEV void stream(const ExpertArgs& g, Jobs& jobs, Place&& locate, const Out& out, uint16_t* lds) {
  typedef Operand<kAKN, S::BM, S::kWaves> OpA;
  typedef Operand<kBKN, S::BN, S::kWaves> OpB;
  constexpr int kCopies = OpA::kCopies + OpB::kCopies;
  constexpr uint32_t kStageBytes = S::kStageElems * 2;
  const int wave = uniform(threadIdx.x >> 6), across = wave % (S::BN / S::WN), down = wave / (S::BN / S::WN);
  OpA A;
  OpB B;
  A.init(g.lda, lds);
  B.init(g.ldb, lds + OpA::kElems);

  // the tile being copied, its next stage, and how many tiles were before it
  Span ia, ib;
  int copying = 0, at = 0, rows, cols;
  int64_t out0;
  // job i that has work, from i on: its place and its operands; false: no more
  auto take = [&](int& i, Span& a, Span& b, int& r, int& c, int64_t& o) {
    for (;; ++i) {
      const Job j = jobs.get(i);
      if (j.expert < 0) return false;
      if (j.first == j.last) continue;
      locate(j, a, b, r, c, o);
      r = uniform(r), c = uniform(c);
      a.fix(), b.fix();
      return true;
    }
  };
  if (!take(copying, ia, ib, rows, cols, out0)) return;
  int here = copying, n = ia.stages, buf = 0;   // the tile being multiplied, its stages, the stage's buffer

  auto advance = [&]() {     // past the stage whose copies were issued
    at = uniform(at + 1);
    if (at < ia.stages) return;
    at = 0, ++copying;
    int r, c;
    int64_t o;
    if (take(copying, ia, ib, r, c, o)) return;
    ia.left = ib.left = 0, ia.stages = INT32_MAX;   // nothing from here on
  };
  auto tail_at = [&]() { return at == ia.stages - 1 ? ia.tail : kDepth; };
#pragma unroll
  for (int h = 0; h < S::kStages; ++h) {
    const u32x4 ba = A.buffer(ia, at), bb = B.buffer(ib, at);
    const int tail = tail_at();
#pragma unroll
    for (int i = 0; i < OpA::kCopies; ++i) A.copy(ba, i, h * kStageBytes, tail);
#pragma unroll
    for (int i = 0; i < OpB::kCopies; ++i) B.copy(bb, i, h * kStageBytes, tail);
    advance();
  }
  wait_copies<kCopies*(S::kStages - 1)>();
  barrier();

  constexpr int kStores = Out::template stores<S>();   // of a wave and whole tile
  bool fresh = false;                // such a tile was written since the last stage
  // a tile of up to kHigh rows: its waves take kWM rows each
  auto tile = [&](auto high_c) {
    constexpr int kHigh = decltype(high_c)::value, kWM = kHigh / (S::BM / S::WM);
    constexpr int FA = kWM / 16, FB = S::WN / 16, kMM = FA * FB;
    const int wm = down * kWM, wn = across * S::WN;
    f32x4 acc[FA][FB];
#pragma unroll
    for (int i = 0; i < FA; ++i)
#pragma unroll
      for (int j = 0; j < FB; ++j) acc[i][j] = f32x4{};
    typename Out::template Rows<FA> known;
    out.load(known, out0, wm + (lane_id() & 15), rows);
    u32x4 fa[FA], fb[2][FB];
    auto frag_a = [&](const uint16_t* st, int s, int i) { fa[i] = OpA::frag(st, wm + 16 * i, s); };
    auto frag_b = [&](const uint16_t* st, int s, int i) { fb[s][i] = OpB::frag(st + OpA::kElems, wn + 16 * i, s); };
#pragma unroll
    for (int i = 0; i < FA; ++i) frag_a(lds + buf * S::kStageElems, 0, i);
#pragma unroll
    for (int i = 0; i < FB; ++i) frag_b(lds + buf * S::kStageElems, 0, i);
    // Blocks are computed transposed: a lane has four consecutive columns of a row.  Step 0 reads the fragments of step 1,
    // step 1 those of the next stage, from the barrier after kHold products on.
    constexpr int kHold = FA >= 4 ? 2 * FB : 0;
    static_assert(kMM - kHold >= FB + kHold / FB || kHold == 0, "a read after each product");
    auto mm = [&](int s, int j) {
      acc[j / FB][j % FB] = mfma16<DT>(fb[s][j % FB], fa[j / FB], acc[j / FB][j % FB]);
      __builtin_amdgcn_sched_barrier(0);
    };
    for (int h = 0; h < n; ++h) {
      const int after = uniform(buf + 1 == S::kStages ? 0 : buf + 1);
      const uint16_t *st = lds + buf * S::kStageElems, *next = lds + after * S::kStageElems;
#pragma unroll
      for (int j = 0; j < kMM; ++j) {
        mm(0, j);
        if (j < FB) frag_b(st, 1, j);
        if (j % FB == FB - 1) frag_a(st, 1, j / FB);
        __builtin_amdgcn_sched_barrier(0);
      }
      const u32x4 ba = A.buffer(ia, at), bb = B.buffer(ib, at);
      const int tail = tail_at();
      // the next stage has landed; those after it may be on their way, and behind them the stores of the tile before
      // (memory operations are counted off in their order)
      auto landed = [&]() {
        if (fresh) wait_copies<kCopies*(S::kStages - 2) + kStores>();
        else wait_copies<kCopies*(S::kStages - 2)>();
        fresh = false;
        if (h == 0) known.arrived();   // waited for here, and not in the end behind the copies of then
        barrier();
        __builtin_amdgcn_sched_barrier(0);
      };
      if (kHold == 0) landed();
#pragma unroll
      for (int j = 0; j < kMM; ++j) {
        mm(1, j);
        if (j == kHold - 1) landed();
        // (the last stage's reads of the next fragments are of no use)
        const int q = j - kHold;
        if (q >= 0) {
          if (q < FB) frag_b(next, 0, q);
          if (q >= FB && q - FB < kHold / FB) frag_a(next, 0, q - FB);
          if (j % FB == FB - 1) frag_a(next, 0, j / FB);
#pragma unroll
          for (int i = 0; i < kCopies; ++i)
            if ((kMM - kHold >= 2 * kCopies ? 2 * i + 1 : i * (kMM - kHold) / kCopies) == q) {
              if (i < OpA::kCopies) A.copy(ba, i, buf * kStageBytes, tail);
              else B.copy(bb, i - OpA::kCopies, buf * kStageBytes, tail);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      advance();
      buf = after;
    }
    out.template write<S, kWM>(g, acc, known, lds, down, across, rows, cols, out0);
    fresh = kHigh == S::BM && rows >= S::BM && cols >= S::BN;
  };

  for (;;) {
    if constexpr (kHalves) {
      if (rows <= S::BM / 4 && S::WM >= 64) tile(std::integral_constant<int, (S::WM >= 64 ? S::BM / 4 : S::BM)>());
      else if (rows <= S::BM / 2) tile(std::integral_constant<int, S::BM / 2>());
      else tile(std::integral_constant<int, S::BM>());
    } else {
      tile(std::integral_constant<int, S::BM>());
    }
    Span a, b;
    ++here;
    if (!take(here, a, b, rows, cols, out0)) break;
    n = a.stages;
  }
  wait_copies<0>();   // none lands in LDS that another workgroup has by then
}

// Zeros in the gradients of the experts without rows, in pieces of 16 K elements: piece p of them all goes to
// workgroup p modulo the grid
template <int OD> APEXW_DEV void zero_weights(const ExpertArgs& g) {
  constexpr int kPiece = 16384, V = OD == APEXW_F32 ? 4 : 8;
  const int64_t per = (int64_t)g.n * g.k, pieces = (per + kPiece - 1) / kPiece;
  int64_t before = 0, p = blockIdx.x;
  int row = 0, begin, end;
  for (int e0 = 0; e0 < g.experts; e0 += 64) {
    look(g, e0, row, begin, end);
    const uint64_t none = __ballot(begin == end && e0 + lane_id() < g.experts);
    const int64_t upto = before + __builtin_popcountll(none) * pieces;
    for (; p < upto; p += gridDim.x) {
      uint64_t left = none;
      for (int64_t skip = (p - before) / pieces; skip > 0; --skip) left &= left - 1;
      const int64_t at = (e0 + __builtin_ctzll(left)) * per, i0 = (p - before) % pieces * kPiece;
      const int n = (int)(per - i0 < kPiece ? per - i0 : kPiece);
      for (int i = threadIdx.x * V; i < n; i += blockDim.x * V) {
        const int64_t o = at + i0 + i;
        if (i + V <= n) {
          if constexpr (OD == APEXW_F32) APEXW_GLOBAL(Chunk32, (float*)g.out + o)->v = u32x4{0u, 0u, 0u, 0u};
          else APEXW_GLOBAL(Chunk, (uint16_t*)g.out + o)->v = u32x4{0u, 0u, 0u, 0u};
        } else {
          for (int j = i; j < n; ++j) store_elem<OD>(g.out, at + i0 + j, 0.0f);
        }
      }
    }
    before = upto;
  }
}

// The sum of n partial sums, in their order
APEXW_DEV float join(const float* p, int64_t stride, int n) {
  float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  int i = 0;
  for (; i + 4 <= n; i += 4)
#pragma unroll
    for (int j = 0; j < 4; ++j) s[j] += p[(i + j) * stride];
  for (; i < n; ++i) s[0] += p[i * stride];
  return (s[0] + s[1]) + (s[2] + s[3]);
}

// Rows of `width` elements, ld apart, groups of `high` of them `step` apart, copied to rows of whole chunks with
// zeros behind their end: what the asynchronous copies need of an operand of another width or address.  Bound by
// bytes, both operands in one launch: 4096 rows of 500 and 8 x 386 more 7 us, most of it the launch.
struct Pad {
  const uint16_t* src;
  int64_t ld, step, high, rows;
  int32_t width;
  u32x4* dst;
};

// I: the index type; 32-bit quotients where all chunks are counted in 32 bits
template <class I> APEXW_DEV void pad_rows(const Pad& p, unsigned group, unsigned groups) {
  const I per = (I)((p.width + 7) / 8), high = (I)p.high, n = (I)p.rows * per, stride = (I)groups * 256;
  for (I i = (I)group * 256 + threadIdx.x; i < n; i += stride) {
    const I row = i / per, c = i - row * per, group = row / high;
    p.dst[i] = load_chunk(p.src + (int64_t)group * p.step + (int64_t)(row - group * high) * p.ld + (int64_t)c * 8,
                          clamp8(p.width - (int64_t)c * 8));
  }
}
__global__ __launch_bounds__(256) void pad_kernel(Pad a, Pad b) {
  const Pad& p = blockIdx.y ? b : a;
  if (p.rows * ((p.width + 7) / 8) < (1ll << 31)) pad_rows<uint32_t>(p, blockIdx.x, gridDim.x);
  else pad_rows<uint64_t>(p, blockIdx.x, gridDim.x);
}

// the most elements from row to row: a stage's copies reach 256 rows by 32-bit byte offsets
constexpr int64_t kMostLd = 1 << 22;

// rows of whole 16-byte chunks at 16-byte addresses, within the offsets of a stage's copies
bool chunks_ok(const void* p, int64_t ld, int64_t width, int64_t step = 0) {
  return ((uintptr_t)p & 15u) == 0 && ld % 8 == 0 && width % 8 == 0 && step % 8 == 0 && ld <= kMostLd;
}
// rows of `width` elements may be copied to whole chunks: the copy's rows, `width` rounded up apart, keep to that
bool copy_ok(int64_t width) { return width <= kMostLd; }
// The same of an operand given as k rows.  Overlapping ones (a row broadcast, sliding windows) would have what lies
// behind the last k row within their memory, so they are copied or go to the general kernel, which tests k.
// (Testing k in each copy instead: dense 8192^3 weight gradient 851 -> 864 us, rows' gradient 878 -> 889 us.)
bool k_rows_ok(const void* p, int64_t ld, int64_t width, int64_t step = 0) {
  return chunks_ok(p, ld, width, step) && ld >= width;
}

// workgroups of a stream: as many as the chip holds at a time, and no more than there are tiles
template <class S> unsigned stream_grid(int64_t tiles) {
  const int64_t most = (int64_t)apexw_cu_count() * S::kPerCU;
  return (unsigned)(((tiles < most ? tiles : most) + 7) / 8 * 8);
}

template <class S> int64_t rows_tiles(const ExpertArgs& g) {
  return (g.rows / S::BM + (g.rows < g.experts ? g.rows : g.experts)) * ((g.n + S::BN - 1) / S::BN);
}
template <class S> int64_t weight_tiles(const ExpertArgs& g) {
  return (int64_t)((g.n + S::BM - 1) / S::BM) * ((g.k + S::BN - 1) / S::BN) * g.experts;
}

// How a product is cut: the shape of its tiles (0: 32 x 128, 1: 64 x 128, 2: 128 x 256, 3: 256 x 256) and the
// parts of what it sums over, chosen for the least time by what a stage takes with every workgroup of the chip
// at work and with few: 256 x 256 1.75 and 0.95 us, 128 x 256 1.0 and 0.65, 64 x 128 0.72 and 0.45, 32 x 128
// 0.55 and 0.42 (from products of 64 to 4096 rows with 4096 x 4096 weights).  An expert's last tile is taken as
// half full.  Measured by shape, the smallest first: 4096 rows of one expert 287, 188, 133, 121 us; 1024 rows
// 76, 51, 59, 94; 64 rows 32, 34, 46, 64; 8192 rows in 8 experts of 2048 x 2048 180, 121, 94, 95; 512 rows in 16
// experts of 4096 x 2048 63, 80, 70, 102.  Parts cost a launch that joins them and 8 bytes an element each, and
// have to gain a fifth (decode steps are soon bound by the weights' bytes): 64 rows of one expert 16 us in
// eight parts, 32 whole; 128 rows over 16 experts of 4096 x 2048 54 in two, 62; 48 rows over 64 experts of
// 2048 x 1024 23.0 in two, 22.4 whole.
struct Cut {
  int shape, splits;
  float cost;
};
template <class S> void try_cut(Cut& best, int shape, float tiles, float stages, float elems, float most, float least,
                                bool may_split) {
  const float slots = (float)(apexw_cu_count() * S::kPerCU);
  for (int n = 1; n == 1 || (may_split && n <= 64 && (float)(4 * n) <= stages && tiles * (float)n <= 1.5f * slots); n *= 2) {
    const float rounds = tiles * (float)n / slots;
    const float stage = rounds <= 1.0f ? least + (most - least) * rounds : most * ceilf(4.0f * rounds) * 0.25f;
    const float cost = n == 1 ? stages * stage : 1.25f * (ceilf(stages / (float)n) * stage + 5.0f + (float)n * elems * 8.0f / 3e6f);
    if (best.splits == 0 || cost < best.cost) best = {shape, n, cost};
  }
}

Cut cut_rows(const ExpertArgs& g, bool may_split) {
  Cut best{0, 0, 0.0f};
  const float used = (float)(g.rows < g.experts ? g.rows : g.experts), stages = (float)((g.wide + 63) / 64);
  const float elems = (float)g.rows * (float)g.n;
  auto tiles = [&](int bm, int bn) {
    const float high = g.experts == 1 ? (float)((g.rows + bm - 1) / bm) : (float)g.rows / (float)bm + 0.5f * used;
    return high * (float)((g.n + bn - 1) / bn);
  };
  try_cut<Small>(best, 0, tiles(32, 128), stages, elems, 0.55f, 0.42f, may_split);
  try_cut<Mid>(best, 1, tiles(64, 128), stages, elems, 0.72f, 0.45f, may_split);
  try_cut<Wide>(best, 2, tiles(128, 256), stages, elems, 1.0f, 0.65f, false);
  try_cut<Large>(best, 3, tiles(256, 256), stages, elems, 1.75f, 0.95f, false);
  return best;
}

// The longest expert counts, which the host does not know: twice the average.  6772 rows over 3 experts of
// 448 x 704, even and uneven: in parts 27 and 32 us, whole 40 and 68.
Cut cut_weight(const ExpertArgs& g, bool may_split) {
  Cut best{0, 0, 0.0f};
  const float uneven = 2.0f * (float)g.rows / (float)g.experts;
  const float stages = ceilf((uneven < (float)g.rows ? uneven : (float)g.rows) / 64.0f) + 1.0f;
  const float elems = (float)g.experts * (float)g.n * (float)g.k;
  try_cut<Wide>(best, 2, (float)weight_tiles<Wide>(g), stages, elems, 1.0f, 0.65f, may_split);
  try_cut<Large>(best, 3, (float)weight_tiles<Large>(g), stages, elems, 1.75f, 0.95f, may_split);
  return best;
}

// a product over k cut into `splits` parts of whole stages, or fewer
void cut_up(ExpertArgs& g, int splits, int stage) {
  if (splits <= 1) return;
  const int32_t stages = (g.wide + stage - 1) / stage;
  g.part = (stages + splits - 1) / splits * stage;
  g.splits = (g.wide + g.part - 1) / g.part;
}
int64_t padded(int64_t rows, int64_t width) { return rows * ((width + 7) / 8 * 8) * 2; }

// An operand to be copied to `at` as rows of whole chunks: advances `at`, replaces address and strides
Pad pad(const uint16_t*& p, int64_t& ld, int64_t& step, int64_t high, int64_t rows, int32_t width, uint16_t*& at) {
  const int64_t wide = (width + 7) / 8 * 8;
  const Pad job{p, ld, step, high, rows, width, (u32x4*)at};
  p = at, ld = wide, step = high * wide;
  at += rows * wide;
  return job;
}
void launch_pad(const Pad& a, const Pad& b, hipStream_t s) {
  const int64_t most = (a.rows * a.width > b.rows * b.width ? a.rows * a.width : b.rows * b.width) / 2048 + 1;
  hipLaunchKernelGGL(pad_kernel, dim3((unsigned)(most < 8192 ? most : 8192), b.rows ? 2 : 1), dim3(256), 0, s, a, b);
}

}  // namespace
