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
#include "tiles.h"

namespace {

constexpr int kTile = 128, kBK = 32;
// LDS elements of one operand's stage: [128 rows][32 k], rows of 80 bytes, or [32 k][128 columns], rows of 272
constexpr int kLdK = 40, kLdN = 136, kStage = kTile * kLdK > kBK * kLdN ? kTile * kLdK : kBK * kLdN;

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

template <class S, bool kBKN, int DT, int OD>
__global__ __launch_bounds__(S::kThreads, 2) void expert_rows_stream_kernel(ExpertArgs g) {
  __shared__ __attribute__((aligned(16))) uint16_t lds[S::kLds];
  RowJobs<true> jobs(g, S::BM, S::BN);
  if (OD != APEXW_F32 && g.which != kRest) zero_rows(g, jobs.rows);
  stream<S, false, kBKN, DT, true>(g, jobs, [&](const Job& j, Span& a, Span& b, int& rows, int& cols, int64_t& out0) {
    const int64_t row = j.first + j.row, col = j.col * S::BN;
    const int k0 = j.split * g.part, wide = g.wide - k0 < g.part ? g.wide - k0 : g.part;
    const int deep = g.k - k0 < g.part ? g.k - k0 : g.part;
    rows = j.last - (int)row, cols = g.n - (int)col, out0 = j.split * g.split_stride + row * g.ldo + col;
    a.set<false>(g.a + row * g.lda + k0, g.lda, rows, wide, S::BM);
    // whole chunks of columns: rows of another width have been copied to such
    b.set<kBKN>(g.b + j.expert * g.sb + (kBKN ? k0 * g.ldb + col : col * g.ldb + k0), g.ldb,
                kBKN ? (cols + 7) / 8 * 8 : cols, kBKN ? deep : wide, S::BN);
  }, Store<OD>(), lds);
}

template <class S, int DT, int OD>
__global__ __launch_bounds__(S::kThreads, 2) void expert_weight_stream_kernel(ExpertArgs g) {
  __shared__ __attribute__((aligned(16))) uint16_t lds[S::kLds];
  if (g.splits == 1) zero_weights<OD>(g);
  WeightJobs jobs(g, S::BM, S::BN);
  stream<S, true, true, DT, false>(g, jobs, [&](const Job& j, Span& a, Span& b, int& rows, int& cols, int64_t& out0) {
    const int64_t row = j.row, col = j.col * S::BN, first = j.first;
    rows = g.n - (int)row, cols = g.k - (int)col;
    out0 = j.split * g.split_stride + (j.expert * (int64_t)g.n + row) * g.k + col;
    a.set<true>(g.a + first * g.lda + row, g.lda, (rows + 7) / 8 * 8, j.last - j.first, S::BM);
    b.set<true>(g.b + first * g.ldb + col, g.ldb, (cols + 7) / 8 * 8, j.last - j.first, S::BN);
  }, Store<OD>(), lds);
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

template <class S, int DT, int OD> void launch_rows(const ExpertArgs& g, bool kn, hipStream_t s) {
  const dim3 grid(stream_grid<S>(rows_tiles<S>(g) * g.splits)), block(S::kThreads);
  if (kn) hipLaunchKernelGGL((expert_rows_stream_kernel<S, true, DT, OD>), grid, block, 0, s, g);
  else hipLaunchKernelGGL((expert_rows_stream_kernel<S, false, DT, OD>), grid, block, 0, s, g);
}
template <class S, int DT, int OD> void launch_weight(const ExpertArgs& g, hipStream_t s) {
  const dim3 grid(stream_grid<S>(weight_tiles<S>(g) * g.splits)), block(S::kThreads);
  hipLaunchKernelGGL((expert_weight_stream_kernel<S, DT, OD>), grid, block, 0, s, g);
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
