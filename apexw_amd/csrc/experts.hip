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
  int64_t first, last, tile;  // its rows, and which of its row tiles
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

// The group (an expert, or the rows behind the last end) that row tile t of `size` rows belongs to.
APEXW_DEV Group find_group(const ExpertArgs& g, int64_t t, int size) {
  int64_t row = 0, tiles = 0;   // the end of the groups before, and their tiles
  for (int e0 = 0; e0 <= g.experts; e0 += 64) {
    const int e = e0 + lane_id();
    int64_t end = e < g.experts ? (int64_t)g.ends[e] : g.rows;
    end = end > g.rows ? g.rows : end < row ? row : end;
    end = wave_prefix_max(end);
    int64_t begin = __shfl_up(end, 1, 64);
    if (lane_id() == 0) begin = row;
    const int64_t mine = e <= g.experts ? (end - begin + size - 1) / size : 0;
    const int64_t upto = tiles + wave_prefix_sum(mine);
    const uint64_t hit = __ballot(t < upto);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      return {e0 + l, __shfl(begin, l, 64), __shfl(end, l, 64), t - __shfl(upto - mine, l, 64)};
    }
    row = __shfl(end, 63, 64);
    tiles = __shfl(upto, 63, 64);
  }
  return {-1, 0, 0, 0};
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
  const Group at = find_group(g, blockIdx.x / cols, kTile);
  if (at.expert < 0) return;
  const int64_t row = at.first + at.tile * kTile, col = (int64_t)(blockIdx.x % cols) * kTile;
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
  const dim3 grid((unsigned)tiles), block(256);
  hipStream_t s = (hipStream_t)stream;
  const bool kn = w_order == APEXW_EXPERT_KN;
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
  if (dtype == APEXW_BF16) {
    if (dw_dtype == APEXW_F32) hipLaunchKernelGGL((expert_weight_kernel<APEXW_BF16, APEXW_F32>), grid, block, 0, s, g);
    else hipLaunchKernelGGL((expert_weight_kernel<APEXW_BF16, APEXW_BF16>), grid, block, 0, s, g);
  } else {
    if (dw_dtype == APEXW_F32) hipLaunchKernelGGL((expert_weight_kernel<APEXW_F16, APEXW_F32>), grid, block, 0, s, g);
    else hipLaunchKernelGGL((expert_weight_kernel<APEXW_F16, APEXW_F16>), grid, block, 0, s, g);
  }
  return hipGetLastError() == hipSuccess ? APEXW_OK : APEXW_ERR_LAUNCH;
}
