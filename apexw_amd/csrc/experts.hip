// Matrix products grouped by expert, with ragged numbers of rows (gfx950).
//
// The rows of a buffer are sorted by expert; ends[e] (device memory) is one past expert e's last row:
//   rows product:  o_i = W_e a_i       the layer's output (W_e [n x k]) or its rows' gradient (W_e^T)
//   weight grad:   dW_e = sum over e's rows of dy_i x_i^T
// 16-bit operands, products on the matrix cores, fp32 accumulation, one rounding at the end.
//
// The number of rows of an expert is known on the device alone.  A launch has as many workgroups as tiles
// could exist (an expert adds at most one partly filled tile); each finds its tile from the ends, those
// without one return.  Ends that decrease or pass the buffer count as clamped, so no access leaves it.
#include <type_traits>

#include "common.h"

namespace {

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(16))) float f32x16;
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
};

struct Group {
  int expert;                 // the number of experts: rows that belong to none; -1: no tile
  int64_t first, last, tile;  // its rows, and which of its tiles
};

APEXW_DEV int64_t wave_prefix_max(int64_t x) {
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int64_t y = __shfl_up(x, off, 64);
    if (lane_id() >= off && y > x) x = y;
  }
  return x;
}
APEXW_DEV int64_t wave_prefix_sum(int64_t x) {
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int64_t y = __shfl_up(x, off, 64);
    if (lane_id() >= off) x += y;
  }
  return x;
}

// One wave's look at 64 groups from e0 on: lane l gets the rows [begin, end) of group e0 + l and the row tiles
// of `size` rows up to and with it; row, tiles: the end of the groups before e0, and their tiles.
APEXW_DEV void look(const ExpertArgs& g, int e0, int size, int64_t& row, int64_t& tiles, int64_t& begin, int64_t& end,
                    int64_t& mine, int64_t& upto) {
  const int e = e0 + lane_id();
  end = e < g.experts ? (int64_t)g.ends[e] : g.rows;
  end = end > g.rows ? g.rows : end < row ? row : end;
  end = wave_prefix_max(end);
  begin = __shfl_up(end, 1, 64);
  if (lane_id() == 0) begin = row;
  mine = e <= g.experts ? (end - begin + size - 1) / size : 0;
  upto = tiles + wave_prefix_sum(mine);
  row = __shfl(end, 63, 64);
  tiles = __shfl(upto, 63, 64);
}

// The workgroup's group (an expert, or the rows behind the last end) and tile of it, of `cols` tiles to a row
// of tiles.  Workgroups go to the 8 XCDs in turn: each XCD gets a contiguous part of the tiles, so that
// those that share rows and weights share its L2.
APEXW_DEV Group find_group(const ExpertArgs& g, int size, int cols) {
  int64_t row = 0, tiles = 0, begin, end, mine, upto;
  look(g, 0, size, row, tiles, begin, end, mine, upto);
  for (int e0 = 64; e0 <= g.experts; e0 += 64) look(g, e0, size, row, tiles, begin, end, mine, upto);
  const int64_t all = tiles * cols, part = (all + 7) / 8, in = blockIdx.x / 8, t = (blockIdx.x % 8) * part + in;
  if (in >= part || t >= all) return {-1, 0, 0, 0};
  if (g.experts >= 64) row = tiles = 0;
  for (int e0 = 0; e0 <= g.experts; e0 += 64) {
    if (g.experts >= 64) look(g, e0, size, row, tiles, begin, end, mine, upto);
    const uint64_t hit = __ballot(t < upto * cols);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      return {e0 + l, __shfl(begin, l, 64), __shfl(end, l, 64), t - __shfl(upto - mine, l, 64) * cols};
    }
  }
  return {-1, 0, 0, 0};
}

// Tile (row, column) of index t among rows x cols tiles: bands of 8 tile rows, column by column
APEXW_DEV void place(int64_t t, int64_t rows, int cols, int64_t& r, int64_t& c) {
  const int64_t band = t / (8 * cols), in = t - band * 8 * cols;
  const int64_t high = rows - band * 8 < 8 ? rows - band * 8 : 8;
  c = in / high;
  r = band * 8 + in - c * high;
}

// the rows of expert e
APEXW_DEV void expert_rows(const ExpertArgs& g, int e, int64_t& first, int64_t& last) {
  first = last = 0;
  for (int e0 = 0; e0 <= e; e0 += 64) {
    const int i = e0 + lane_id();
    int64_t x = i <= e ? (int64_t)g.ends[i] : 0, y = i < e ? x : 0;
    x = x > g.rows ? g.rows : x < 0 ? 0 : x;
    y = y > g.rows ? g.rows : y < 0 ? 0 : y;
    x = __shfl(wave_prefix_max(x), 63, 64);
    y = __shfl(wave_prefix_max(y), 63, 64);
    first = y > first ? y : first;
    last = x > last ? x : last;
  }
}

struct __attribute__((packed, aligned(2))) Chunk { u32x4 v; };

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
// base: row 0, k 0 (row stride ld); rows / depth: how many of them there are.
template <bool kKN>
APEXW_DEV void fetch(const uint16_t* base, int64_t ld, int64_t rows, int64_t depth, int64_t k0, u32x4 (&r)[2]) {
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

// One operand of a tile: `kSize` of its rows (or, kKN, columns) over the k of a stage.
//   k-contiguous: LDS [kSize rows][64 k]; the 8 chunks of row r are swapped by XOR with (r / 2) % 8, so that the
//     fragment reads of 16 consecutive rows touch every bank once
//   kKN: LDS [64 k][kSize columns]; the chunks of k row r are swapped by XOR with 4 (r % 4), so that the
//     transposing reads of 4 consecutive k rows do
template <bool kKN, int kSize, int kWaves> struct Operand {
  static constexpr int kElems = kSize * kDepth;            // of a stage
  static constexpr int kCopies = kSize / 8 / kWaves;       // 1 KB each
  const uint16_t* base;
  int64_t step, left;     // bytes from stage to stage, and from the base to the operand's end
  uint32_t voff[kCopies]; // per lane
  uint32_t lds0;          // of this wave's first copy in stage 0
  int tail;               // k-contiguous: k of the last stage that this lane's chunks must stay below

  // base: row (column) 0, k 0; ld: elements from row to row (k row to k row); rows: rows (columns) that
  // exist; depth: k that exist; width: elements of a memory row from the base on (kKN: columns that exist)
  __device__ __forceinline__ void init(const uint16_t* p, int64_t ld, int64_t rows, int64_t depth, const uint16_t* lds) {
    const int lane = lane_id(), wave = threadIdx.x >> 6;
    base = p;
    step = (kKN ? (int64_t)kDepth * ld : kDepth) * 2;
    left = kKN ? ((depth - 1) * ld + rows) * 2 : (((rows < kSize ? rows : kSize) - 1) * ld + depth) * 2;
    tail = (int)((depth - 1) % kDepth) + 1;
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
      const int q = wave * kCopies + i;
      if constexpr (kKN) {
        constexpr int kChunks = kSize / 8;
        const int k = q * (64 / kChunks) + lane / kChunks, chunk = (lane % kChunks) ^ (4 * (k & 3));
        voff[i] = (uint32_t)(k * ld + chunk * 8) * 2u;
      } else {
        const int row = q * 8 + (lane >> 3);
        voff[i] = (uint32_t)(row * ld + chunk_of(i) * 8) * 2u;
      }
    }
    lds0 = __builtin_amdgcn_readfirstlane(
        (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)(lds + wave * kCopies * 512));
  }
  __device__ __forceinline__ int chunk_of(int i) const {   // k-contiguous: the chunk that this lane's copy i brings
    const int lane = lane_id(), q = (threadIdx.x >> 6) * kCopies + i;
    return (lane & 7) ^ ((4 * (q & 1) + (lane >> 4)) & 7);
  }
  __device__ __forceinline__ u32x4 buffer(int h) const {
    const uint64_t at = (uint64_t)base + (uint64_t)(h * step);
    int64_t n = left - h * step;
    n = n < 0 ? 0 : n > 0xFFFFFF00ll ? 0xFFFFFF00ll : n;
    return u32x4{uniform((uint32_t)at), uniform((uint32_t)(at >> 32)), uniform((uint32_t)n), 0x00020000u};
  }
  // copy i of a stage into the buffer at LDS byte `to`; last: the stage where k may end
  __device__ __forceinline__ void copy(u32x4 b, int i, uint32_t to, bool last) const {
    uint32_t v = voff[i];
    if constexpr (!kKN) v = last && chunk_of(i) * 8 >= tail ? kNowhere : v;
    lds_copy16(lds0 + to + i * 1024, v, b);
  }
  // the fragment of 32 rows (columns) from `row` at k step s
  static __device__ __forceinline__ u32x4 frag(const uint16_t* lds, int row, int s) {
    const int lane = lane_id();
    if constexpr (kKN) {
      const int g = lane >> 4, r = lane & 3, jr = (lane >> 2) & 3;
      const int n = row + 16 * (g & 1) + 4 * r, k = 16 * s + 8 * (g >> 1) + jr;
      const int e = k * kSize + (((n >> 3) ^ (4 * jr)) << 3) + (n & 7);
      const v4i16 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4i16*)&lds[e]);
      const v4i16 hi =
          __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4i16*)&lds[e + 4 * kSize]);
      const u32x2 wl = __builtin_bit_cast(u32x2, lo), wh = __builtin_bit_cast(u32x2, hi);
      return u32x4{wl[0], wl[1], wh[0], wh[1]};
    } else {
      const int r = row + (lane & 31), c = (2 * s + (lane >> 5)) ^ ((lane >> 1) & 7);   // row: a multiple of 32
      return *(const u32x4*)&lds[r * kDepth + c * 8];
    }
  }
};

// A tile's shape: BM x BN by waves of WM x WN, kStages stages of 64 k in LDS
template <int BM_, int BN_, int WM_, int WN_, int kStages_> struct Shape {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, kStages = kStages_;
  static constexpr int kWaves = (BM / WM) * (BN / WN), kThreads = kWaves * 64;
  static constexpr int kStageElems = (BM + BN) * kDepth, kLds = kStages * kStageElems;
};
typedef Shape<256, 256, 128, 64, 2> Large;
typedef Shape<128, 256, 128, 64, 3> Wide;

// One tile of A B^T: `rows` x `cols` of it exist, over `depth` > 0.  In a stage's four k steps each MFMA is
// followed by at most one fragment read of the next step and one copy, fenced in place: issued in bursts they
// stall the wave's in-order issue.  The barrier stands before the last step, whose fragments are in registers
// by then: behind it the stage's buffer is free for the copies of kStages stages on, and the next stage,
// landed, gives its first fragments.
template <class S, bool kAKN, bool kBKN, int DT, int OD>
APEXW_DEV void fast_tile(const uint16_t* a, int64_t lda, const uint16_t* b, int64_t ldb, int64_t rows, int64_t cols,
                         int64_t depth, void* out, int64_t out0, int64_t ldo, uint16_t* lds) {
  constexpr int FA = S::WM / 32, FB = S::WN / 32, kFrags = FA + FB, kMM = FA * FB;
  typedef Operand<kAKN, S::BM, S::kWaves> OpA;
  typedef Operand<kBKN, S::BN, S::kWaves> OpB;
  constexpr int kCopies = OpA::kCopies + OpB::kCopies;
  constexpr uint32_t kStageBytes = S::kStageElems * 2;
  // 16-bit results leave through LDS by rows: their blocks are computed transposed (four consecutive columns
  // to a lane); fp32 ones leave as they are (32 lanes, 32 columns)
  constexpr bool kSwap = OD != APEXW_F32;
  const int lane = lane_id(), wave = threadIdx.x >> 6;
  const int wm = wave / (S::BN / S::WN) * S::WM, wn = wave % (S::BN / S::WN) * S::WN;
  OpA A;
  OpB B;
  A.init(a, lda, rows, depth, lds);
  B.init(b, ldb, cols, depth, lds + OpA::kElems);
  const int n = (int)((depth + kDepth - 1) / kDepth);

  f32x16 acc[FA][FB];
#pragma unroll
  for (int i = 0; i < FA; ++i)
#pragma unroll
    for (int j = 0; j < FB; ++j) acc[i][j] = f32x16{};
  u32x4 fa[2][FA], fb[2][FB];
  auto frag = [&](const uint16_t* st, int s, int i) {
    if (i < FA) fa[s & 1][i] = OpA::frag(st, wm + 32 * i, s);
    else fb[s & 1][i - FA] = OpB::frag(st + OpA::kElems, wn + 32 * (i - FA), s);
  };
  auto step = [&](int s, auto&& side) {
#pragma unroll
    for (int j = 0; j < kMM; ++j) {
      const int x = j / FB, y = j % FB;
      if constexpr (kSwap) acc[x][y] = mfma<DT>(fb[s & 1][y], fa[s & 1][x], acc[x][y]);
      else acc[x][y] = mfma<DT>(fa[s & 1][x], fb[s & 1][y], acc[x][y]);
      __builtin_amdgcn_sched_barrier(0);
      side(j);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  const int first = n < S::kStages ? n : S::kStages;
  for (int h = 0; h < first; ++h) {
    const u32x4 ba = A.buffer(h), bb = B.buffer(h);
#pragma unroll
    for (int i = 0; i < OpA::kCopies; ++i) A.copy(ba, i, h * kStageBytes, h == n - 1);
#pragma unroll
    for (int i = 0; i < OpB::kCopies; ++i) B.copy(bb, i, h * kStageBytes, h == n - 1);
  }
  if (first == S::kStages) wait_copies<kCopies*(S::kStages - 1)>();
  else wait_copies<0>();
  barrier();
#pragma unroll
  for (int i = 0; i < kFrags; ++i) frag(lds, 0, i);

  // kRefill: stage h + kStages exists; kNext: stage h + 1 does
  auto stage = [&](int h, int buf, auto refill_c, auto next_c) {
    constexpr bool kRefill = decltype(refill_c)::value, kNext = decltype(next_c)::value;
    const uint16_t* st = lds + buf * S::kStageElems;
    const int next = buf + 1 == S::kStages ? 0 : buf + 1;
#pragma unroll
    for (int s = 0; s < 3; ++s)
      step(s, [&](int j) {
        if (j < kFrags) frag(st, s + 1, j);
      });
    // stage h + 1 has landed; those after it may be on their way
    if constexpr (kRefill) wait_copies<kCopies*(S::kStages - 2)>();
    else wait_copies<0>();
    barrier();
    u32x4 ba{}, bb{};
    bool last = false;
    if constexpr (kRefill) {
      ba = A.buffer(h + S::kStages);
      bb = B.buffer(h + S::kStages);
      last = h + S::kStages == n - 1;
    }
    step(3, [&](int j) {
      if constexpr (kNext) {
        if (j < kFrags) frag(lds + next * S::kStageElems, 0, j);
      }
      if constexpr (kRefill) {
#pragma unroll
        for (int i = j * kCopies / kMM; i < (j + 1) * kCopies / kMM; ++i) {
          if (i < OpA::kCopies) A.copy(ba, i, buf * kStageBytes, last);
          else B.copy(bb, i - OpA::kCopies, buf * kStageBytes, last);
        }
      }
    });
  };
  typedef std::integral_constant<bool, true> yes;
  typedef std::integral_constant<bool, false> no;
  int h = 0, buf = 0;
  for (; h + S::kStages < n; ++h) {
    stage(h, buf, yes(), yes());
    buf = buf + 1 == S::kStages ? 0 : buf + 1;
  }
  for (; h + 1 < n; ++h) {
    stage(h, buf, no(), yes());
    buf = buf + 1 == S::kStages ? 0 : buf + 1;
  }
  stage(h, buf, no(), no());

  if constexpr (kSwap) {
    // lane l has row l % 32, columns 8 (q / 4) + 4 (l / 32) + q % 4 of a block.  Each wave puts its block into
    // LDS of its own (the operands there are dead behind the last barrier) in rows of WN, chunks swapped by
    // XOR with the row, and writes it out in whole lines.
    static_assert(S::WN == 64, "rows of 8 chunks");
    uint16_t* mine = lds + wave * S::WM * S::WN;
#pragma unroll
    for (int i = 0; i < FA; ++i)
#pragma unroll
      for (int j = 0; j < FB; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int r = 32 * i + (lane & 31), c = 4 * j + q;
          const f32x16& v = acc[i][j];
          u32x2 w;
          if constexpr (OD == APEXW_BF16)
            w = u32x2{pack_bf16x2(v[4 * q], v[4 * q + 1]), pack_bf16x2(v[4 * q + 2], v[4 * q + 3])};
          else
            w = u32x2{f32_to_f16_bits(v[4 * q]) | (f32_to_f16_bits(v[4 * q + 1]) << 16),
                      f32_to_f16_bits(v[4 * q + 2]) | (f32_to_f16_bits(v[4 * q + 3]) << 16)};
          *(u32x2*)&mine[r * 64 + ((c ^ (r & 7)) << 3) + 4 * (lane >> 5)] = w;
        }
#pragma unroll 4
    for (int i = 0; i < S::WM / 8; ++i) {
      const int r = 8 * i + (lane >> 3), c = lane & 7;
      const u32x4 w = *(const u32x4*)&mine[r * 64 + ((c ^ (r & 7)) << 3)];
      if (wm + r < rows && wn + 8 * c < cols)
        *APEXW_GLOBAL(u32x4, (uint16_t*)out + out0 + (wm + r) * ldo + wn + 8 * c) = w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < FA; ++i)
#pragma unroll
      for (int j = 0; j < FB; ++j)
#pragma unroll
        for (int q = 0; q < 16; ++q) {
          const int r = wm + 32 * i + 8 * (q >> 2) + 4 * (lane >> 5) + (q & 3), c = wn + 32 * j + (lane & 31);
          if (r < rows && c < cols) APEXW_GLOBAL(float, out)[out0 + r * ldo + c] = acc[i][j][q];
        }
  }
}

// Zeros for rows that belong to no expert
template <class S> APEXW_DEV void zero_tile(void* out, int64_t out0, int64_t ldo, int64_t rows, int64_t cols) {
  for (int c = threadIdx.x; c < S::BM * S::BN / 8; c += S::kThreads) {
    const int r = c / (S::BN / 8), e = c % (S::BN / 8) * 8;
    if (r < rows && e < cols) *APEXW_GLOBAL(u32x4, (uint16_t*)out + out0 + r * ldo + e) = u32x4{0u, 0u, 0u, 0u};
  }
}

template <class S, bool kBKN, int DT>
__global__ __launch_bounds__(S::kThreads, S::kWaves / 4) void expert_rows_fast_kernel(ExpertArgs g) {
  __shared__ __attribute__((aligned(16))) uint16_t lds[S::kLds];
  const int cols = (g.n + S::BN - 1) / S::BN;
  const Group at = find_group(g, S::BM, cols);
  if (at.expert < 0) return;
  int64_t row, col;
  place(at.tile, (at.last - at.first + S::BM - 1) / S::BM, cols, row, col);
  row = at.first + row * S::BM, col *= S::BN;
  if (at.expert == g.experts) {
    zero_tile<S>(g.out, row * g.ldo + col, g.ldo, at.last - row, g.n - col);
    return;
  }
  const uint16_t* w = g.b + at.expert * g.sb + (kBKN ? col : col * g.ldb);
  fast_tile<S, false, kBKN, DT, DT>(g.a + row * g.lda, g.lda, w, g.ldb, at.last - row, g.n - col, g.k, g.out,
                                    row * g.ldo + col, g.ldo, lds);
}

template <class S, int DT, int OD>
__global__ __launch_bounds__(S::kThreads, S::kWaves / 4) void expert_weight_fast_kernel(ExpertArgs g) {
  __shared__ __attribute__((aligned(16))) uint16_t lds[S::kLds];
  const int tn = (g.n + S::BM - 1) / S::BM, tk = (g.k + S::BN - 1) / S::BN, per = tn * tk;
  // each XCD takes a contiguous part of every expert's tiles: experts differ in rows, and so in work
  const int part = (per + 7) / 8, i = blockIdx.x / 8, e = i / part, t = (blockIdx.x % 8) * part + i % part;
  if (t >= per) return;
  int64_t row, col, first, last;
  place(t, tn, tk, row, col);
  row *= S::BM, col *= S::BN;
  expert_rows(g, e, first, last);
  const int64_t at = ((int64_t)e * g.n + row) * g.k + col;
  if (first == last) {
    for (int c = threadIdx.x; c < S::BM * S::BN / 4; c += S::kThreads) {
      const int r = c / (S::BN / 4), x = c % (S::BN / 4) * 4;
      if (row + r < g.n && col + x < g.k) {
        if constexpr (OD == APEXW_F32) *APEXW_GLOBAL(u32x4, (float*)g.out + at + (int64_t)r * g.k + x) = u32x4{0u, 0u, 0u, 0u};
        else *APEXW_GLOBAL(u32x2, (uint16_t*)g.out + at + (int64_t)r * g.k + x) = u32x2{0u, 0u};
      }
    }
    return;
  }
  fast_tile<S, true, true, DT, OD>(g.a + first * g.lda + row, g.lda, g.b + first * g.ldb + col, g.ldb, g.n - row,
                                   g.k - col, last - first, g.out, at, g.k, lds);
}

// ---------------------------------------------------------------------------
// Any alignment
// ---------------------------------------------------------------------------

// One 128 x 128 tile of A B^T: `rows` x `cols` of it exist, over `depth`.  Four waves of 64 x 64, a stage of
// 32 k in registers while the one before is multiplied.
template <bool kAKN, bool kBKN, int DT, int OD>
APEXW_DEV void tile(const uint16_t* a, int64_t lda, const uint16_t* b, int64_t ldb, int64_t rows, int64_t cols,
                    int64_t depth, void* out, int64_t out0, int64_t ldo) {
  __shared__ __attribute__((aligned(16))) uint16_t lds[2][2][kStage];
  const int lane = lane_id(), wave = threadIdx.x >> 6, wm = (wave >> 1) * 64, wn = (wave & 1) * 64;
  f32x16 acc[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) acc[i][j] = f32x16{};
  u32x4 ra[2], rb[2];
  if (depth > 0) {
    fetch<kAKN>(a, lda, rows, depth, 0, ra);
    fetch<kBKN>(b, ldb, cols, depth, 0, rb);
  }
  int p = 0;
  for (int64_t k0 = 0; k0 < depth; k0 += kBK, p ^= 1) {
    put<kAKN>(lds[p][0], ra);
    put<kBKN>(lds[p][1], rb);
    __syncthreads();
    if (k0 + kBK < depth) {
      fetch<kAKN>(a, lda, rows, depth, k0 + kBK, ra);
      fetch<kBKN>(b, ldb, cols, depth, k0 + kBK, rb);
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

template <bool kBKN, int DT>
__global__ __launch_bounds__(256) void expert_rows_kernel(ExpertArgs g) {
  const int cols = (g.n + kTile - 1) / kTile;
  const Group at = find_group(g, kTile, cols);
  if (at.expert < 0) return;
  int64_t row, col;
  place(at.tile, (at.last - at.first + kTile - 1) / kTile, cols, row, col);
  row = at.first + row * kTile, col *= kTile;
  const bool none = at.expert == g.experts;
  const uint16_t* w = g.b + (none ? 0 : at.expert * g.sb) + (kBKN ? col : col * g.ldb);
  tile<false, kBKN, DT, DT>(g.a + row * g.lda, g.lda, w, g.ldb, at.last - row, g.n - col, none ? 0 : g.k, g.out,
                            row * g.ldo + col, g.ldo);
}

template <int DT, int OD>
__global__ __launch_bounds__(256) void expert_weight_kernel(ExpertArgs g) {
  const int tn = (g.n + kTile - 1) / kTile, tk = (g.k + kTile - 1) / kTile;
  const int e = blockIdx.x / (tn * tk), t = blockIdx.x % (tn * tk);
  const int64_t row = (int64_t)(t / tk) * kTile, col = (int64_t)(t % tk) * kTile;
  int64_t first, last;
  expert_rows(g, e, first, last);
  tile<true, true, DT, OD>(g.a + first * g.lda + row, g.lda, g.b + first * g.ldb + col, g.ldb, g.n - row, g.k - col,
                           last - first, g.out, ((int64_t)e * g.n + row) * g.k + col, g.k);
}

// rows of whole 16-byte chunks at 16-byte addresses, within the 32-bit offsets of a stage's copies
bool chunks_ok(const void* p, int64_t ld, int64_t width, int64_t step = 0) {
  return ((uintptr_t)p & 15u) == 0 && ld % 8 == 0 && width % 8 == 0 && step % 8 == 0 && ld <= (1 << 22);
}

template <class S, int DT>
void launch_rows(const ExpertArgs& g, bool kn, int64_t tiles, hipStream_t s) {
  const dim3 grid((unsigned)((tiles + 7) / 8 * 8)), block(S::kThreads);
  if (kn) hipLaunchKernelGGL((expert_rows_fast_kernel<S, true, DT>), grid, block, 0, s, g);
  else hipLaunchKernelGGL((expert_rows_fast_kernel<S, false, DT>), grid, block, 0, s, g);
}

template <class S, int DT>
void launch_weight(const ExpertArgs& g, int32_t out_dtype, hipStream_t s) {
  const int64_t per = (int64_t)((g.n + S::BM - 1) / S::BM) * ((g.k + S::BN - 1) / S::BN);
  const dim3 grid((unsigned)((per + 7) / 8 * 8 * g.experts)), block(S::kThreads);
  if (out_dtype == APEXW_F32) hipLaunchKernelGGL((expert_weight_fast_kernel<S, DT, APEXW_F32>), grid, block, 0, s, g);
  else hipLaunchKernelGGL((expert_weight_fast_kernel<S, DT, DT>), grid, block, 0, s, g);
}

bool sizes_ok(int64_t rows, int32_t experts, int64_t n, int64_t k) {
  return rows >= 0 && rows <= INT32_MAX && experts > 0 && n > 0 && k > 0 && n <= INT32_MAX - 256 && k <= INT32_MAX - 256;
}

}  // namespace

extern "C" int apexw_expert_rows(const void* a, int64_t lda, const void* w, int64_t w_row_stride, int64_t w_expert_stride,
                                 int32_t w_order, const int32_t* ends, int32_t experts, int64_t rows, int64_t k,
                                 int64_t n, int32_t dtype, void* out, int64_t ldo, void* stream) {
  if (!a || !w || !ends || !out || !sizes_ok(rows, experts, n, k)) return APEXW_ERR_ARG;
  if (lda < 0 || w_row_stride < 0 || w_expert_stride < 0 || ldo < n) return APEXW_ERR_ARG;
  if (w_order != APEXW_EXPERT_NK && w_order != APEXW_EXPERT_KN) return APEXW_ERR_ARG;
  if (dtype != APEXW_BF16 && dtype != APEXW_F16) return APEXW_ERR_DTYPE;
  if (((uintptr_t)a | (uintptr_t)w | (uintptr_t)out) & 1u || (uintptr_t)ends & 3u) return APEXW_ERR_ALIGN;
  if (rows == 0) return APEXW_OK;
  const int64_t tiles = (rows / kTile + (rows < experts + 1 ? rows : experts + 1)) * ((n + kTile - 1) / kTile);
  if (tiles > INT32_MAX) return APEXW_ERR_SIZE;
  ExpertArgs g{(const uint16_t*)a, (const uint16_t*)w, ends, out, lda, w_row_stride, w_expert_stride, ldo, rows,
               experts, (int32_t)n, (int32_t)k};
  const dim3 grid((unsigned)((tiles + 7) / 8 * 8)), block(256);
  hipStream_t s = (hipStream_t)stream;
  const bool kn = w_order == APEXW_EXPERT_KN;
  if (chunks_ok(a, lda, k) && chunks_ok(w, w_row_stride, kn ? n : k, w_expert_stride) && chunks_ok(out, ldo, n)) {
    auto most = [&](int bm, int bn) {
      return (rows / bm + (rows < experts + 1 ? rows : experts + 1)) * ((n + bn - 1) / bn);
    };
    const bool large = rows >= (int64_t)experts * 512;
    const int64_t count = large ? most(Large::BM, Large::BN) : most(Wide::BM, Wide::BN);
    if (dtype == APEXW_BF16) {
      if (large) launch_rows<Large, APEXW_BF16>(g, kn, count, s);
      else launch_rows<Wide, APEXW_BF16>(g, kn, count, s);
    } else {
      if (large) launch_rows<Large, APEXW_F16>(g, kn, count, s);
      else launch_rows<Wide, APEXW_F16>(g, kn, count, s);
    }
    return hipGetLastError() == hipSuccess ? APEXW_OK : APEXW_ERR_LAUNCH;
  }
  if (dtype == APEXW_BF16) {
    if (kn) hipLaunchKernelGGL((expert_rows_kernel<true, APEXW_BF16>), grid, block, 0, s, g);
    else hipLaunchKernelGGL((expert_rows_kernel<false, APEXW_BF16>), grid, block, 0, s, g);
  } else {
    if (kn) hipLaunchKernelGGL((expert_rows_kernel<true, APEXW_F16>), grid, block, 0, s, g);
    else hipLaunchKernelGGL((expert_rows_kernel<false, APEXW_F16>), grid, block, 0, s, g);
  }
  return hipGetLastError() == hipSuccess ? APEXW_OK : APEXW_ERR_LAUNCH;
}

extern "C" int apexw_expert_weight_grad(const void* dy, int64_t ld_dy, const void* x, int64_t ld_x, const int32_t* ends,
                                        int32_t experts, int64_t rows, int64_t n, int64_t k, int32_t dtype, void* dw,
                                        int32_t dw_dtype, void* stream) {
  if (!ends || !dw || !sizes_ok(rows, experts, n, k) || (rows > 0 && (!dy || !x))) return APEXW_ERR_ARG;
  if (ld_dy < 0 || ld_x < 0) return APEXW_ERR_ARG;
  if ((dtype != APEXW_BF16 && dtype != APEXW_F16) || (dw_dtype != dtype && dw_dtype != APEXW_F32)) return APEXW_ERR_DTYPE;
  if (((uintptr_t)dy | (uintptr_t)x) & 1u || (uintptr_t)ends & 3u || (uintptr_t)dw & (dw_dtype == APEXW_F32 ? 3u : 1u))
    return APEXW_ERR_ALIGN;
  const int64_t tiles = (int64_t)experts * ((n + kTile - 1) / kTile) * ((k + kTile - 1) / kTile);
  if (tiles > INT32_MAX) return APEXW_ERR_SIZE;
  ExpertArgs g{(const uint16_t*)dy, (const uint16_t*)x, ends, dw, ld_dy, ld_x, 0, k, rows, experts, (int32_t)n,
               (int32_t)k};
  const dim3 grid((unsigned)tiles), block(256);
  hipStream_t s = (hipStream_t)stream;
  if (chunks_ok(dy, ld_dy, n) && chunks_ok(x, ld_x, k) && chunks_ok(dw, k, k)) {
    if (dtype == APEXW_BF16) launch_weight<Large, APEXW_BF16>(g, dw_dtype, s);
    else launch_weight<Large, APEXW_F16>(g, dw_dtype, s);
    return hipGetLastError() == hipSuccess ? APEXW_OK : APEXW_ERR_LAUNCH;
  }
  if (dtype == APEXW_BF16) {
    if (dw_dtype == APEXW_F32) hipLaunchKernelGGL((expert_weight_kernel<APEXW_BF16, APEXW_F32>), grid, block, 0, s, g);
    else hipLaunchKernelGGL((expert_weight_kernel<APEXW_BF16, APEXW_BF16>), grid, block, 0, s, g);
  } else {
    if (dw_dtype == APEXW_F32) hipLaunchKernelGGL((expert_weight_kernel<APEXW_F16, APEXW_F32>), grid, block, 0, s, g);
    else hipLaunchKernelGGL((expert_weight_kernel<APEXW_F16, APEXW_F16>), grid, block, 0, s, g);
  }
  return hipGetLastError() == hipSuccess ? APEXW_OK : APEXW_ERR_LAUNCH;
}
