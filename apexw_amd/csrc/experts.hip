// Matrix products grouped by expert, with ragged numbers of rows (gfx950).
//
// The rows of a buffer are sorted by expert; ends[e] (device memory) is one past expert e's last row:
//   rows product:  o_i = W_e a_i       the layer's output (W_e [n x k]) or its rows' gradient (W_e^T)
//   weight grad:   dW_e = sum over e's rows of dy_i x_i^T
// 16-bit operands, products on the matrix cores, fp32 accumulation, one rounding at the end.
//
// The number of rows of an expert is known on the device alone: each workgroup finds its tiles from the ends.
// Ends that decrease or pass the buffer count as clamped, so no access leaves it.
//
// Measured (bf16, random normal operands; a library's product of one matrix of the first size takes 1360 us):
//   output, 8 experts of 14336 x 4096, 16384 rows           1770 us   1090 TFLOP/s
//   the same, one expert                                     1500 us   1280 TFLOP/s
//   rows' gradient, 32 uneven experts of 2048 x 4096, 8192   204 us    670 TFLOP/s, 3.1 TB/s
//   weights' gradient in fp32, 16 of 4096 x 2048, 16384      336 us    820 TFLOP/s, 2.2 TB/s
//   48 rows over 64 experts of 1024 x 2048                   22.4 us   4.7 TB/s of weights
// Dense products of 8192^3 run at 1280 (rows along k), 1250 and 1270 TFLOP/s: the chip's power bounds them, at
// 1.8 GHz and two thirds of the matrix cores' cycles.  Without its MFMAs a stage of a 256 x 256 tile still
// takes 85% of its time, waiting for its 64 KB from L2, which is why tiles of few rows gain little.
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

constexpr int kTile = 128, kBK = 32;
// LDS elements of one operand's stage: [128 rows][32 k], rows of 80 bytes, or [32 k][128 columns], rows of 272
constexpr int kLdK = 40, kLdN = 136, kStage = kTile * kLdK > kBK * kLdN ? kTile * kLdK : kBK * kLdN;

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

// A stage of one operand in registers: 128 rows x 32 k, kKN: given as k rows of 128 columns.
// base: row 0, k 0 (row stride ld); rows / depth: how many of them there are; before: how many columns of a
// kKN operand's rows stand ahead of base.  A whole stage loads without a branch, the last row again in place of
// rows that do not exist: what they give is not stored.  Of a tile that ends inside a chunk, the row's last 8
// elements are loaded in the chunk's place and shifted: 1 row of 7578 elements with an expert of 7578 x 387
// 286 us with the tail's elements one by one.
template <bool kKN>
APEXW_DEV void fetch(const uint16_t* base, int64_t ld, int64_t rows, int64_t depth, int64_t k0, u32x4 (&r)[2],
                     int64_t before = 0) {
  if (kKN && k0 + kBK <= depth && rows < kTile && before + rows >= 8) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int c = threadIdx.x + 256 * i, col = (c & 15) * 8, at = col + 8 <= (int)rows ? col : (int)rows - 8;
      const u32x4 v = APEXW_GLOBAL(const Chunk, base + (k0 + (c >> 4)) * ld + at)->v;
      const int bits = col - at < 8 ? 16 * (col - at) : 0;   // 0: behind the last column, whatever it holds
      const uint64_t lo = (uint64_t)v[1] << 32 | v[0], hi = (uint64_t)v[3] << 32 | v[2];
      const uint64_t up = bits == 0 ? 0 : bits < 64 ? hi << (64 - bits) : hi >> (bits - 64);
      const uint64_t l = bits < 64 ? lo >> bits | up : up, h = bits < 64 ? hi >> bits : 0;
      r[i] = u32x4{(uint32_t)l, (uint32_t)(l >> 32), (uint32_t)h, (uint32_t)(h >> 32)};
    }
    return;
  }
  if (k0 + kBK <= depth && (!kKN || rows >= kTile)) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int c = threadIdx.x + 256 * i;
      const int64_t row = (c >> 2) < rows ? c >> 2 : rows - 1;
      const uint16_t* p = kKN ? base + (k0 + (c >> 4)) * ld + (c & 15) * 8 : base + row * ld + k0 + (c & 3) * 8;
      r[i] = APEXW_GLOBAL(const Chunk, p)->v;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int c = threadIdx.x + 256 * i;
    if constexpr (kKN) {
      const int64_t k = k0 + (c >> 4);
      const int col = (c & 15) * 8;
      r[i] = load_chunk(base + k * ld + col, k < depth ? clamp8(rows - col) : 0);
    } else {
      const int row = c >> 2;
      const int64_t k = k0 + (c & 3) * 8;
      r[i] = load_chunk(base + row * ld + k, row < rows ? clamp8(depth - k) : 0);
    }
  }
}
template <bool kKN> APEXW_DEV void put(uint16_t* lds, const u32x4 (&r)[2]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int c = threadIdx.x + 256 * i;
    *(u32x4*)&lds[kKN ? (c >> 4) * kLdN + (c & 15) * 8 : (c >> 2) * kLdK + (c & 3) * 8] = r[i];
  }
}

// Fragment of 32 rows from `row` at k step s (16 k): lane l has row l % 32, k = 8 (l / 32) .. + 7.
// From [k][column] by two transposing reads: in each 16 lanes, lane 4 r + c gets element c of the 8-byte
// rows that lanes r, r + 4, r + 8, r + 12 address.
template <bool kKN> APEXW_DEV u32x4 fragment(const uint16_t* lds, int row, int s) {
  const int lane = lane_id();
  if constexpr (kKN) {
    const int g = lane >> 4, r = lane & 3, jr = (lane >> 2) & 3;
    const int e = (16 * s + 8 * (g >> 1) + jr) * kLdN + row + 16 * (g & 1) + 4 * r;
    const v4i16 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4i16*)&lds[e]);
    const v4i16 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4i16*)&lds[e + 4 * kLdN]);
    const u32x2 wl = __builtin_bit_cast(u32x2, lo), wh = __builtin_bit_cast(u32x2, hi);
    return u32x4{wl[0], wl[1], wh[0], wh[1]};
  } else {
    return *(const u32x4*)&lds[(row + (lane & 31)) * kLdK + 16 * s + 8 * (lane >> 5)];
  }
}

template <int DT> APEXW_DEV f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (DT == APEXW_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

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

// zeros in the rows from `row` on, which belong to no expert
APEXW_DEV void zero_rows(const ExpertArgs& g, int row) {
  const bool vec = g.n % 8 == 0;
  const int V = vec ? 8 : 1;
  const int64_t per = g.n / V, n = (g.rows - row) * per, step = (int64_t)gridDim.x * blockDim.x;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += step) {
    uint16_t* p = (uint16_t*)g.out + (row + i / per) * g.ldo + i % per * V;
    if (vec) APEXW_GLOBAL(Chunk, p)->v = u32x4{0u, 0u, 0u, 0u};
    else *APEXW_GLOBAL(uint16_t, p) = 0;
  }
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

// The tiles of a workgroup, each A B^T over its k, as one stream of stages: the copies of a tile's first
// stages are under way while the tile before is multiplied and written out.
//
// A stage is two steps of 32 k by 16 x 16 x 32 MFMAs (at the power limit, which bounds large products of real
// numbers, they reach 2160 TFLOP/s from registers where 32 x 32 x 16 ones reach 1950).  After an MFMA come at
// most one fragment read of the next step and one copy, fenced in place: issued in bursts they stall the
// wave's in-order issue.  The barrier stands between the steps, when the second one's fragments are in
// registers: behind it the stage's buffer is free for the copies of the stage kStages on, and the next stage,
// landed, gives its first fragments.  A's fragments are read into the registers of the ones just used.
template <class S, bool kAKN, bool kBKN, int DT, int OD, bool kHalves, class Jobs, class Place>
APEXW_DEV void stream(const ExpertArgs& g, Jobs& jobs, Place&& locate, uint16_t* lds) {
  typedef Operand<kAKN, S::BM, S::kWaves> OpA;
  typedef Operand<kBKN, S::BN, S::kWaves> OpB;
  constexpr int kCopies = OpA::kCopies + OpB::kCopies;
  constexpr uint32_t kStageBytes = S::kStageElems * 2;
  const int wave = uniform(threadIdx.x >> 6), across = wave % (S::BN / S::WN), down = wave / (S::BN / S::WN);
  uint16_t* mine = lds + S::kStages * S::kStageElems + wave * S::kOut;
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
  bool more = take(copying, ia, ib, rows, cols, out0);
  if (!more) return;
  int here = copying, n = ia.stages, buf = 0;   // the tile being multiplied, its stages, the stage's buffer

  auto advance = [&]() {     // past the stage whose copies were issued
    at = uniform(at + 1);
    if (at < ia.stages) return;
    at = 0, ++copying;
    int r, c;
    int64_t o;
    more = take(copying, ia, ib, r, c, o);
  };
  int ready = 0;             // stages in flight at the start
  for (; ready < S::kStages && more; ++ready) {
    const u32x4 ba = A.buffer(ia, at), bb = B.buffer(ib, at);
    const int tail = at == ia.stages - 1 ? ia.tail : kDepth;
#pragma unroll
    for (int i = 0; i < OpA::kCopies; ++i) A.copy(ba, i, ready * kStageBytes, tail);
#pragma unroll
    for (int i = 0; i < OpB::kCopies; ++i) B.copy(bb, i, ready * kStageBytes, tail);
    advance();
  }

  bool full = ready == S::kStages;   // the copies of the stage kStages - 1 on are under way
  if (full) wait_copies<kCopies*(S::kStages - 1)>();
  else wait_copies<0>();
  barrier();

  constexpr int kStores = S::WM / 16 * (S::WN * (OD == APEXW_F32 ? 4 : 2) / 64);   // of a wave and whole tile
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
    u32x4 fa[FA], fb[2][FB];
    auto frag_a = [&](const uint16_t* st, int s, int i) { fa[i] = OpA::frag(st, wm + 16 * i, s); };
    auto frag_b = [&](const uint16_t* st, int s, int i) { fb[s][i] = OpB::frag(st + OpA::kElems, wn + 16 * i, s); };
#pragma unroll
    for (int i = 0; i < FA; ++i) frag_a(lds + buf * S::kStageElems, 0, i);
#pragma unroll
    for (int i = 0; i < FB; ++i) frag_b(lds + buf * S::kStageElems, 0, i);
    // step s; blocks are computed transposed: a lane has four consecutive columns of a row.  Step s1 of the stage
    // at st1 is next; side: what else is issued
    auto step = [&](int s, const uint16_t* st1, int s1, auto&& side) {
#pragma unroll
      for (int j = 0; j < kMM; ++j) {
        const int x = j / FB, y = j % FB;
        acc[x][y] = mfma16<DT>(fb[s][y], fa[x], acc[x][y]);
        __builtin_amdgcn_sched_barrier(0);
        if (j < FB) frag_b(st1, s1, j);
        if (y == FB - 1) frag_a(st1, s1, x);
        side(j);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    for (int h = 0; h < n; ++h) {
      const uint16_t* st = lds + buf * S::kStageElems;
      const int after = uniform(buf + 1 == S::kStages ? 0 : buf + 1);
      step(0, st, 1, [](int) {});
      // the next stage has landed; those after it may be on their way, and behind them the stores of the tile
      // before (memory operations are counted off in their order)
      if (fresh) {
        if (full) wait_copies<kCopies*(S::kStages - 2) + kStores>();
        else wait_copies<kStores>();
        fresh = false;
      } else {
        if (full) wait_copies<kCopies*(S::kStages - 2)>();
        else wait_copies<0>();
      }
      barrier();
      const bool refill = more;
      const u32x4 ba = A.buffer(ia, at), bb = B.buffer(ib, at);   // (of no use without a stage to copy)
      const int tail = at == ia.stages - 1 ? ia.tail : kDepth;
      // (the last stage's reads of the next fragments are of no use)
      step(1, lds + after * S::kStageElems, 0, [&](int j) {
        if (refill) {
#pragma unroll
          for (int i = 0; i < kCopies; ++i)
            if ((kMM >= 2 * kCopies ? 2 * i + 1 : i * kMM / kCopies) == j) {
              if (i < OpA::kCopies) A.copy(ba, i, buf * kStageBytes, tail);
              else B.copy(bb, i - OpA::kCopies, buf * kStageBytes, tail);
            }
        }
      });
      if (refill) advance();
      full = refill;
      buf = after;
    }
    // Write the tile out: lane l has row l % 16, columns 4 (l / 16) .. + 3 of a block.  Each wave puts 16 rows of
    // 128 bytes into LDS of its own, chunks swapped by XOR with the row, and writes them out in whole lines.
    // (Addresses are formed here, not kept in registers over the stages.)
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
          const f32x4 v = acc[i][j0 + j];
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
          const u32x4 w = *(const u32x4*)&mine[(r * kChunks + (c ^ (r & (kChunks - 1)))) * 8];
          const int row = wm + 16 * i + r, col = wn + 16 * j0 + kPer * c;
          if (row >= rows || col >= cols) continue;
          const int64_t o = out0 + row * g.ldo + col;
          if (col + kPer <= cols) {   // at any element address: rows of odd width start anywhere
            if constexpr (OD == APEXW_F32) APEXW_GLOBAL(Chunk32, (float*)g.out + o)->v = w;
            else APEXW_GLOBAL(Chunk, (uint16_t*)g.out + o)->v = w;
          } else {
#pragma unroll
            for (int x = 0; x < kPer; ++x)
              if (col + x < cols) {
                if constexpr (OD == APEXW_F32) APEXW_GLOBAL(uint32_t, g.out)[o + x] = w[x];
                else APEXW_GLOBAL(uint16_t, g.out)[o + x] = (uint16_t)(w[x >> 1] >> (16 * (x & 1)));
              }
          }
        }
      }
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
    if (!take(here, a, b, rows, cols, out0)) return;
    n = a.stages;
  }
}

template <class S, bool kBKN, int DT, int OD>
__global__ __launch_bounds__(S::kThreads, 2) void expert_rows_stream_kernel(ExpertArgs g) {
  __shared__ __attribute__((aligned(16))) uint16_t lds[S::kLds];
  RowJobs<true> jobs(g, S::BM, S::BN);
  if (OD != APEXW_F32 && g.which != kRest) zero_rows(g, jobs.rows);
  stream<S, false, kBKN, DT, OD, true>(g, jobs, [&](const Job& j, Span& a, Span& b, int& rows, int& cols, int64_t& out0) {
    const int64_t row = j.first + j.row, col = j.col * S::BN;
    const int k0 = j.split * g.part, wide = g.wide - k0 < g.part ? g.wide - k0 : g.part;
    const int deep = g.k - k0 < g.part ? g.k - k0 : g.part;
    rows = j.last - (int)row, cols = g.n - (int)col, out0 = j.split * g.split_stride + row * g.ldo + col;
    a.set<false>(g.a + row * g.lda + k0, g.lda, rows, wide, S::BM);
    // whole chunks of columns: rows of another width have been copied to such
    b.set<kBKN>(g.b + j.expert * g.sb + (kBKN ? k0 * g.ldb + col : col * g.ldb + k0), g.ldb,
                kBKN ? (cols + 7) / 8 * 8 : cols, kBKN ? deep : wide, S::BN);
  }, lds);
}

template <class S, int DT, int OD>
__global__ __launch_bounds__(S::kThreads, 2) void expert_weight_stream_kernel(ExpertArgs g) {
  __shared__ __attribute__((aligned(16))) uint16_t lds[S::kLds];
  if (g.splits == 1) zero_weights<OD>(g);
  WeightJobs jobs(g, S::BM, S::BN);
  stream<S, true, true, DT, OD, false>(g, jobs, [&](const Job& j, Span& a, Span& b, int& rows, int& cols, int64_t& out0) {
    const int64_t row = j.row, col = j.col * S::BN, first = j.first;
    rows = g.n - (int)row, cols = g.k - (int)col;
    out0 = j.split * g.split_stride + (j.expert * (int64_t)g.n + row) * g.k + col;
    a.set<true>(g.a + first * g.lda + row, g.lda, (rows + 7) / 8 * 8, j.last - j.first, S::BM);
    b.set<true>(g.b + first * g.ldb + col, g.ldb, (cols + 7) / 8 * 8, j.last - j.first, S::BN);
  }, lds);
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

// The parts of a rows product added up (partial: [splits][rows][n]); zeros behind the last end
template <int OD> __global__ __launch_bounds__(256) void join_rows_kernel(ExpertArgs g, const float* __restrict__ partial) {
  int row = 0, begin, end;
  for (int e0 = 0; e0 < g.experts; e0 += 64) look(g, e0, row, begin, end);
  const int64_t n = g.rows * g.n, some = (int64_t)row * g.n;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const float x = i < some ? join(partial + i, g.split_stride, g.splits) : 0.0f;
    if (g.ldo == g.n) store_elem<OD>(g.out, i, x);
    else store_elem<OD>(g.out, i / g.n * g.ldo + i % g.n, x);
  }
}

// The parts of a weight grad (partial: [splits][experts][n][k]), blockIdx.y an expert: those that have rows
template <int OD>
__global__ __launch_bounds__(256) void join_weight_kernel(ExpertArgs g, const float* __restrict__ partial) {
  const int64_t per = (int64_t)g.n * g.k;
  for (int e = blockIdx.y; e < g.experts; e += gridDim.y) {
    int row = 0, begin, end;
    for (int e0 = 0; e0 <= e; e0 += 64) look(g, e0, row, begin, end);
    const int rows = lane_of(end, e & 63) - lane_of(begin, e & 63);
    const int parts = rows ? (rows + split_rows(rows, g.splits) - 1) / split_rows(rows, g.splits) : 0;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < per; i += (int64_t)gridDim.x * 256)
      store_elem<OD>(g.out, e * per + i, join(partial + e * per + i, g.split_stride, parts));
  }
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
template <class I> APEXW_DEV void pad_rows(const Pad& p) {
  const I per = (I)((p.width + 7) / 8), high = (I)p.high, n = (I)p.rows * per, stride = (I)gridDim.x * 256;
  for (I i = (I)blockIdx.x * 256 + threadIdx.x; i < n; i += stride) {
    const I row = i / per, c = i - row * per, group = row / high;
    p.dst[i] = load_chunk(p.src + (int64_t)group * p.step + (int64_t)(row - group * high) * p.ld + (int64_t)c * 8,
                          clamp8(p.width - (int64_t)c * 8));
  }
}
__global__ __launch_bounds__(256) void pad_kernel(Pad a, Pad b) {
  const Pad& p = blockIdx.y ? b : a;
  if (p.rows * ((p.width + 7) / 8) < (1ll << 31)) pad_rows<uint32_t>(p);
  else pad_rows<uint64_t>(p);
}

// ---------------------------------------------------------------------------
// Any alignment
// ---------------------------------------------------------------------------

// Elements loaded at their own addresses into registers, put into LDS a stage later.  Each stage waits for its
// loads (0.7 us where few workgroups run), so it is bound by latency and goes to few rows and small products,
// cut into parts: 4096 rows over 8 experts of 386 x 500 17.6 us, 90 TFLOP/s; 8 rows over 46 experts of
// 3686 x 943 32 us (73 whole); long products reach about 380 TFLOP/s.

// One 128 x 128 tile of A B^T: `rows` x `cols` of it exist, over `depth`.  Four waves of 64 x 64, a stage of
// 32 k in registers while the one before is multiplied.
template <bool kAKN, bool kBKN, int DT, int OD>
APEXW_DEV void tile(const uint16_t* a, int64_t lda, const uint16_t* b, int64_t ldb, int64_t rows, int64_t cols,
                    int64_t depth, void* out, int64_t out0, int64_t ldo, int64_t a_before, int64_t b_before) {
  __shared__ __attribute__((aligned(16))) uint16_t lds[2][2][kStage];
  const int lane = lane_id(), wave = threadIdx.x >> 6, wm = (wave >> 1) * 64, wn = (wave & 1) * 64;
  f32x16 acc[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) acc[i][j] = f32x16{};
  u32x4 ra[2], rb[2];
  if (depth > 0) {
    fetch<kAKN>(a, lda, rows, depth, 0, ra, a_before);
    fetch<kBKN>(b, ldb, cols, depth, 0, rb, b_before);
  }
  int p = 0;
  for (int64_t k0 = 0; k0 < depth; k0 += kBK, p ^= 1) {
    put<kAKN>(lds[p][0], ra);
    put<kBKN>(lds[p][1], rb);
    __syncthreads();
    if (k0 + kBK < depth) {
      fetch<kAKN>(a, lda, rows, depth, k0 + kBK, ra, a_before);
      fetch<kBKN>(b, ldb, cols, depth, k0 + kBK, rb, b_before);
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      u32x4 fa[2], fb[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        fa[i] = fragment<kAKN>(lds[p][0], wm + 32 * i, s);
        fb[i] = fragment<kBKN>(lds[p][1], wn + 32 * i, s);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = mfma<DT>(fa[i], fb[j], acc[i][j]);
    }
  }
  // lane l holds column l % 32, rows 8 (q / 4) + 4 (l / 32) + q % 4 for accumulator register q
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int q = 0; q < 16; ++q) {
        const int r = wm + 32 * i + 8 * (q >> 2) + 4 * (lane >> 5) + (q & 3), c = wn + 32 * j + (lane & 31);
        if (r < rows && c < cols) store_elem<OD>(out, out0 + r * ldo + c, acc[i][j][q]);
      }
}

template <bool kBKN, int DT, int OD>
__global__ __launch_bounds__(256) void expert_rows_kernel(ExpertArgs g) {
  RowJobs<false> jobs(g, kTile, kTile);
  if (OD != APEXW_F32) zero_rows(g, jobs.rows);
  const Job j = jobs.get(0);
  if (j.expert < 0) return;
  const int64_t row = j.first + j.row, col = (int64_t)j.col * kTile, k0 = (int64_t)j.split * g.part;
  const uint16_t* w = g.b + j.expert * g.sb + (kBKN ? k0 * g.ldb + col : col * g.ldb + k0);
  tile<false, kBKN, DT, OD>(g.a + row * g.lda + k0, g.lda, w, g.ldb, j.last - row, g.n - col,
                            g.k - k0 < g.part ? g.k - k0 : g.part, g.out, j.split * g.split_stride + row * g.ldo + col,
                            g.ldo, 0, col);
}

template <int DT, int OD>
__global__ __launch_bounds__(256) void expert_weight_kernel(ExpertArgs g) {
  zero_weights<OD>(g);
  const Job j = WeightJobs(g, kTile, kTile).get(0);
  if (j.expert < 0 || j.first == j.last) return;
  const int64_t row = j.row, col = (int64_t)j.col * kTile;
  tile<true, true, DT, OD>(g.a + j.first * g.lda + row, g.lda, g.b + j.first * g.ldb + col, g.ldb, g.n - row, g.k - col,
                           j.last - j.first, g.out, ((int64_t)j.expert * g.n + row) * g.k + col, g.k, row, col);
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

template <class S, int DT, int OD> void launch_rows(const ExpertArgs& g, bool kn, hipStream_t s) {
  const dim3 grid(stream_grid<S>(rows_tiles<S>(g) * g.splits)), block(S::kThreads);
  if (kn) hipLaunchKernelGGL((expert_rows_stream_kernel<S, true, DT, OD>), grid, block, 0, s, g);
  else hipLaunchKernelGGL((expert_rows_stream_kernel<S, false, DT, OD>), grid, block, 0, s, g);
}
template <class S, int DT, int OD> void launch_weight(const ExpertArgs& g, hipStream_t s) {
  const dim3 grid(stream_grid<S>(weight_tiles<S>(g) * g.splits)), block(S::kThreads);
  hipLaunchKernelGGL((expert_weight_stream_kernel<S, DT, OD>), grid, block, 0, s, g);
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

// The general kernel's 128 x 128 tiles, stages of 32 k
struct Any { static constexpr int kPerCU = 2; };
Cut cut_any(const ExpertArgs& g, bool may_split) {
  Cut best{0, 0, 0.0f};
  const float used = (float)(g.rows < g.experts ? g.rows : g.experts);
  const float tiles = ((float)g.rows / kTile + (g.experts == 1 ? 0.5f : used)) * (float)((g.n + kTile - 1) / kTile);
  try_cut<Any>(best, 0, tiles, (float)((g.k + kBK - 1) / kBK), (float)g.rows * (float)g.n, 1.4f, 0.7f, may_split);
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

template <int DT> void launch_rows_as(const ExpertArgs& g, bool kn, int shape, hipStream_t s) {
  if (g.splits > 1) {
    if (shape == 1) launch_rows<Mid, DT, APEXW_F32>(g, kn, s);
    else launch_rows<Small, DT, APEXW_F32>(g, kn, s);
  } else if (shape == 3) {
    ExpertArgs h = g;
    h.which = kMost;
    launch_rows<Large, DT, DT>(h, kn, s);
    h.which = kRest;
    launch_rows<Wide, DT, DT>(h, kn, s);
  } else if (shape == 2) {
    launch_rows<Wide, DT, DT>(g, kn, s);
  } else if (shape == 1) {
    launch_rows<Mid, DT, DT>(g, kn, s);
  } else {
    launch_rows<Small, DT, DT>(g, kn, s);
  }
}
template <int DT, int OD> void launch_weight_to(const ExpertArgs& g, int shape, hipStream_t s) {
  if (shape == 3) launch_weight<Large, DT, OD>(g, s);
  else launch_weight<Wide, DT, OD>(g, s);
}
template <int DT> void launch_weight_as(const ExpertArgs& g, int shape, bool fp32, hipStream_t s) {
  if (fp32 || g.splits > 1) launch_weight_to<DT, APEXW_F32>(g, shape, s);
  else launch_weight_to<DT, DT>(g, shape, s);
}

// f(the type code as a constant) for an output's type
template <class F> void by_type(int32_t dtype, F&& f) {
  if (dtype == APEXW_F32) f(std::integral_constant<int, APEXW_F32>());
  else if (dtype == APEXW_BF16) f(std::integral_constant<int, APEXW_BF16>());
  else f(std::integral_constant<int, APEXW_F16>());
}

// a product over k cut into `splits` parts of whole stages, or fewer
void cut_up(ExpertArgs& g, int splits, int stage) {
  if (splits <= 1) return;
  const int32_t stages = (g.wide + stage - 1) / stage;
  g.part = (stages + splits - 1) / splits * stage;
  g.splits = (g.wide + g.part - 1) / g.part;
}
void launch_join(const ExpertArgs& g, int32_t dtype, const float* partial, hipStream_t s) {
  const int64_t grid = (g.rows * g.n + 255) / 256;
  by_type(dtype, [&](auto d) {
    hipLaunchKernelGGL(join_rows_kernel<decltype(d)::value>, dim3((unsigned)(grid < 4096 ? grid : 4096)), dim3(256), 0, s,
                       g, partial);
  });
}
template <int DT, int OD> void launch_any_to(const ExpertArgs& g, bool kn, hipStream_t s) {
  const int64_t tiles = (g.rows / kTile + (g.rows < g.experts ? g.rows : g.experts)) * ((g.n + kTile - 1) / kTile) * g.splits;
  const dim3 grid((unsigned)((tiles + 7) / 8 * 8)), block(256);
  if (kn) hipLaunchKernelGGL((expert_rows_kernel<true, DT, OD>), grid, block, 0, s, g);
  else hipLaunchKernelGGL((expert_rows_kernel<false, DT, OD>), grid, block, 0, s, g);
}
template <int DT> void launch_any(const ExpertArgs& g, bool kn, hipStream_t s) {
  if (g.splits > 1) launch_any_to<DT, APEXW_F32>(g, kn, s);
  else launch_any_to<DT, DT>(g, kn, s);
}

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

// Operands of other widths are copied where the products gain more by it than the copies take: rows that run
// along k at once in both need many rows an expert (the weights, copied whole, are most of the copies) and long
// sums, weights [k][n], whose rows the general kernel turns around in LDS, fewer.  8 experts, us copied and on
// the general kernel by rows an expert:
//   y = x W^T, 4003 x 2001 weights      64: 80, 70    256: 115, 110   512: 147, 171   2048: 386, 533
//   the same, 1003 x 501                64: 19, 17    256: 23, 20     512: 28, 22     2048: 53, 51
//   dx = dy W, 4003 x 2001              64: 90, 75    128: 99, 126    512: 190, 241   2048: 428, 602
//   the same, 1003 x 501                64: 24, 17    128: 24, 23     512: 29, 51     2048: 56, 61
bool rows_worth_copying(const ExpertArgs& g, bool kn) {
  if (kn) return g.rows >= 96 * (int64_t)g.experts;
  return g.rows >= (g.k >= 1024 ? 384 : 3000) * (int64_t)g.experts;
}
// A weight gradient's operands are small next to its output where rows are few: 8 experts of 4003 x 2001,
// 4 rows each 40, 51; 256 70, 99; of 1003 x 501 4 rows 13.7, 9.9; 256 24.4, 25.4; 16 of 777 x 1531, 12 rows
// 26.7, 22.5.
bool weight_worth_copying(const ExpertArgs& g) {
  return g.rows >= 256 * (int64_t)g.experts || (int64_t)g.experts * g.n >= (1 << 25) / g.k;
}
int64_t padded(int64_t rows, int64_t width) { return rows * ((width + 7) / 8 * 8) * 2; }

// What a call does, and the workspace that it needs: the copies first, the parts' sums behind them
struct Plan {
  bool fast, pad_a, pad_b;
  Cut cut;
  int64_t pads, bytes;
};
Plan plan_rows(ExpertArgs& g, bool kn, bool may) {
  Plan p{};
  const bool fast_a = chunks_ok(g.a, g.lda, g.k);
  const bool fast_w = kn ? k_rows_ok(g.b, g.ldb, g.n, g.sb) : chunks_ok(g.b, g.ldb, g.k, g.sb);
  p.fast = (fast_a && fast_w) || (may && rows_worth_copying(g, kn) && (fast_a || copy_ok(g.k)) &&
                                  (fast_w || copy_ok(kn ? g.n : g.k)));
  if (!p.fast) {
    p.cut = cut_any(g, may);
    p.bytes = p.cut.splits > 1 ? p.cut.splits * g.rows * g.n * 4 : 0;
    return p;
  }
  p.pad_a = !fast_a, p.pad_b = !fast_w;
  if (p.pad_a || p.pad_b) g.wide = (g.k + 7) / 8 * 8;
  p.pads = (p.pad_a ? padded(g.rows, g.k) : 0) + (p.pad_b ? padded(g.experts * (int64_t)(kn ? g.k : g.n), kn ? g.n : g.k) : 0);
  p.cut = cut_rows(g, may);
  p.bytes = p.pads + (p.cut.splits > 1 ? p.cut.splits * g.rows * g.n * 4 : 0);
  return p;
}
Plan plan_weight(ExpertArgs& g, bool may) {
  Plan p{};
  const bool fast_y = k_rows_ok(g.a, g.lda, g.n), fast_x = k_rows_ok(g.b, g.ldb, g.k);
  p.fast = (fast_y && fast_x) ||
           (may && weight_worth_copying(g) && (fast_y || copy_ok(g.n)) && (fast_x || copy_ok(g.k)));
  if (!p.fast) return p;
  p.pad_a = !fast_y, p.pad_b = !fast_x;
  p.pads = (p.pad_a ? padded(g.rows, g.n) : 0) + (p.pad_b ? padded(g.rows, g.k) : 0);
  p.cut = cut_weight(g, may);
  p.bytes = p.pads + (p.cut.splits > 1 ? p.cut.splits * g.split_stride * 4 : 0);
  return p;
}

ExpertArgs rows_args(const void* a, int64_t lda, const void* w, int64_t ldw, int64_t sw, const int32_t* ends, void* out,
                     int64_t ldo, int32_t experts, int64_t rows, int64_t k, int64_t n) {
  return {(const uint16_t*)a, (const uint16_t*)w, ends, out, lda, ldw, sw, ldo, rows, experts, (int32_t)n, (int32_t)k,
          (int32_t)k, 1, INT32_MAX, rows * n, kAll};
}
ExpertArgs weight_args(const void* dy, int64_t ld_dy, const void* x, int64_t ld_x, const int32_t* ends, void* dw,
                       int32_t experts, int64_t rows, int64_t n, int64_t k) {
  return {(const uint16_t*)dy, (const uint16_t*)x, ends, dw, ld_dy, ld_x, 0, k, rows, experts, (int32_t)n, (int32_t)k,
          0, 1, 0, (int64_t)experts * n * k, kAll};
}

bool sizes_ok(int64_t rows, int32_t experts, int64_t n, int64_t k) {
  return rows >= 0 && rows <= INT32_MAX && experts > 0 && n > 0 && k > 0 && n <= INT32_MAX - 256 && k <= INT32_MAX - 256;
}

}  // namespace

extern "C" int64_t apexw_expert_rows_workspace(const void* a, int64_t lda, const void* w, int64_t w_row_stride,
                                               int64_t w_expert_stride, int32_t w_order, int32_t experts, int64_t rows,
                                               int64_t k, int64_t n) {
  if (!sizes_ok(rows, experts, n, k)) return -APEXW_ERR_ARG;
  ExpertArgs g = rows_args(a, lda, w, w_row_stride, w_expert_stride, nullptr, nullptr, n, experts, rows, k, n);
  return plan_rows(g, w_order == APEXW_EXPERT_KN, true).bytes;
}

extern "C" int64_t apexw_expert_weight_grad_workspace(const void* dy, int64_t ld_dy, const void* x, int64_t ld_x,
                                                      int32_t experts, int64_t rows, int64_t n, int64_t k) {
  if (!sizes_ok(rows, experts, n, k)) return -APEXW_ERR_ARG;
  ExpertArgs g = weight_args(dy, ld_dy, x, ld_x, nullptr, nullptr, experts, rows, n, k);
  return plan_weight(g, true).bytes;
}

extern "C" int apexw_expert_rows(const void* a, int64_t lda, const void* w, int64_t w_row_stride, int64_t w_expert_stride,
                                 int32_t w_order, const int32_t* ends, int32_t experts, int64_t rows, int64_t k,
                                 int64_t n, int32_t dtype, void* out, int64_t ldo, void* workspace, void* stream) {
  if (!a || !w || !ends || !out || !sizes_ok(rows, experts, n, k)) return APEXW_ERR_ARG;
  if (lda < 0 || w_row_stride < 0 || w_expert_stride < 0 || ldo < n) return APEXW_ERR_ARG;
  if (w_order != APEXW_EXPERT_NK && w_order != APEXW_EXPERT_KN) return APEXW_ERR_ARG;
  if (dtype != APEXW_BF16 && dtype != APEXW_F16) return APEXW_ERR_DTYPE;
  if (((uintptr_t)a | (uintptr_t)w | (uintptr_t)out) & 1u || (uintptr_t)ends & 3u || (uintptr_t)workspace & 15u)
    return APEXW_ERR_ALIGN;
  if (rows == 0) return APEXW_OK;
  ExpertArgs g = rows_args(a, lda, w, w_row_stride, w_expert_stride, ends, out, ldo, experts, rows, k, n);
  // 32-bit tile counts and rows, with room to round them up
  if (rows > INT32_MAX - 256 || rows_tiles<Small>(g) > INT32_MAX) return APEXW_ERR_SIZE;
  hipStream_t s = (hipStream_t)stream;
  const bool kn = w_order == APEXW_EXPERT_KN;
  const Plan p = plan_rows(g, kn, workspace != nullptr);
  if (p.fast) {
    uint16_t* at = (uint16_t*)workspace;
    int64_t none = 0;
    Pad jobs[2] = {};
    int count = 0;
    if (p.pad_a) jobs[count++] = pad(g.a, g.lda, none, rows, rows, (int32_t)k, at);
    if (p.pad_b) jobs[count++] = pad(g.b, g.ldb, g.sb, kn ? k : n, experts * (kn ? k : n), (int32_t)(kn ? n : k), at);
    if (count) launch_pad(jobs[0], jobs[1], s);
    cut_up(g, p.cut.splits, 64);
    ExpertArgs h = g;
    if (g.splits > 1) h.out = (char*)workspace + p.pads, h.ldo = n;
    if (dtype == APEXW_BF16) launch_rows_as<APEXW_BF16>(h, kn, p.cut.shape, s);
    else launch_rows_as<APEXW_F16>(h, kn, p.cut.shape, s);
    if (g.splits > 1) launch_join(g, dtype, (const float*)h.out, s);
    return hipGetLastError() == hipSuccess ? APEXW_OK : APEXW_ERR_LAUNCH;
  }
  cut_up(g, p.cut.splits, kBK);
  ExpertArgs h = g;
  if (g.splits > 1) h.out = workspace, h.ldo = n;
  if (dtype == APEXW_BF16) launch_any<APEXW_BF16>(h, kn, s);
  else launch_any<APEXW_F16>(h, kn, s);
  if (g.splits > 1) launch_join(g, dtype, (const float*)h.out, s);
  return hipGetLastError() == hipSuccess ? APEXW_OK : APEXW_ERR_LAUNCH;
}

extern "C" int apexw_expert_weight_grad(const void* dy, int64_t ld_dy, const void* x, int64_t ld_x, const int32_t* ends,
                                        int32_t experts, int64_t rows, int64_t n, int64_t k, int32_t dtype, void* dw,
                                        int32_t dw_dtype, void* workspace, void* stream) {
  if (!ends || !dw || !sizes_ok(rows, experts, n, k) || (rows > 0 && (!dy || !x))) return APEXW_ERR_ARG;
  if (ld_dy < 0 || ld_x < 0) return APEXW_ERR_ARG;
  if ((dtype != APEXW_BF16 && dtype != APEXW_F16) || (dw_dtype != dtype && dw_dtype != APEXW_F32)) return APEXW_ERR_DTYPE;
  if (((uintptr_t)dy | (uintptr_t)x) & 1u || (uintptr_t)ends & 3u || (uintptr_t)dw & (dw_dtype == APEXW_F32 ? 3u : 1u) ||
      (uintptr_t)workspace & 15u)
    return APEXW_ERR_ALIGN;
  const int64_t tiles = (((n + kTile - 1) / kTile) * ((k + kTile - 1) / kTile) + 7) / 8 * 8 * experts;
  if (tiles > INT32_MAX || rows > INT32_MAX - 256) return APEXW_ERR_SIZE;
  hipStream_t s = (hipStream_t)stream;
  ExpertArgs g = weight_args(dy, ld_dy, x, ld_x, ends, dw, experts, rows, n, k);
  const Plan p = plan_weight(g, workspace != nullptr);
  if (p.fast) {
    uint16_t* at = (uint16_t*)workspace;
    int64_t none = 0;
    Pad jobs[2] = {};
    int count = 0;
    if (p.pad_a) jobs[count++] = pad(g.a, g.lda, none, rows, rows, (int32_t)n, at);
    if (p.pad_b) jobs[count++] = pad(g.b, g.ldb, none, rows, rows, (int32_t)k, at);
    if (count) launch_pad(jobs[0], jobs[1], s);
    g.splits = p.cut.splits;
    ExpertArgs h = g;
    if (g.splits > 1) h.out = (char*)workspace + p.pads;
    if (dtype == APEXW_BF16) launch_weight_as<APEXW_BF16>(h, p.cut.shape, dw_dtype == APEXW_F32, s);
    else launch_weight_as<APEXW_F16>(h, p.cut.shape, dw_dtype == APEXW_F32, s);
    if (g.splits > 1) {
      const int64_t grid = (n * k + 255) / 256;
      by_type(dw_dtype, [&](auto d) {
        hipLaunchKernelGGL(join_weight_kernel<decltype(d)::value>,
                           dim3((unsigned)(grid < 1024 ? grid : 1024), (unsigned)(experts < 1024 ? experts : 1024)),
                           dim3(256), 0, s, g, (const float*)h.out);
      });
    }
    return hipGetLastError() == hipSuccess ? APEXW_OK : APEXW_ERR_LAUNCH;
  }
  const dim3 grid((unsigned)tiles), block(256);
  if (dtype == APEXW_BF16) {
    if (dw_dtype == APEXW_F32) hipLaunchKernelGGL((expert_weight_kernel<APEXW_BF16, APEXW_F32>), grid, block, 0, s, g);
    else hipLaunchKernelGGL((expert_weight_kernel<APEXW_BF16, APEXW_BF16>), grid, block, 0, s, g);
  } else {
    if (dw_dtype == APEXW_F32) hipLaunchKernelGGL((expert_weight_kernel<APEXW_F16, APEXW_F32>), grid, block, 0, s, g);
    else hipLaunchKernelGGL((expert_weight_kernel<APEXW_F16, APEXW_F16>), grid, block, 0, s, g);
  }
  return hipGetLastError() == hipSuccess ? APEXW_OK : APEXW_ERR_LAUNCH;
}
