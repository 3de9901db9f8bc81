// Softmax cross entropy of a linear head over a large vocabulary, without its logits, and the gradient (gfx950).
//
//   l = x W^T (rows x vocabulary),  lse = log sum_v exp(l_v),  loss = lse - l_target
//   G = (exp(l - lse) - onehot(target)) dloss,  dx = G W,  dW = G^T x
// 16-bit operands, products on the matrix cores, logits and all statistics in fp32.
//
// Rows without a target (ignored, or outside the vocabulary) are left out before anything is multiplied: the rows that
// count are packed together, whole chunks wide, so a masked batch costs what its other rows cost and what stands in
// masked rows, NaN too, reaches nothing.  Their number is known on the device alone.
//
// Forward: the logits of a tile stay in registers, and each row leaves the sum of exponentials over a wave's columns,
// relative to a number near its target's logit, which the packing forms; a second launch joins them.  Backward: a piece
// of the vocabulary at a time, which bounds G's memory; G of the piece from the logits computed again, rounded to 16 bits as
// an operand of the two products that take it: the matrix cores take no other beside 16-bit rows and weights, and a second
// half of G would double the two products.  It is most of what the gradients are off by besides their own rounding (against 64
// bits 0.0019 of the result in bf16 and 0.00025 in fp16, 0.0017 and 0.00021 with G in fp32).  dx adds up the pieces in fp32.
//
// Measured, kernels alone, bf16:
//   forward, 8192 rows, 4096 x 128256       pack 36, logits 6200 to 6370, join 24 us   1350 to 1390 TFLOP/s
//   (a library's product alone 5990 us; the chip's power bounds both)
//   forward, 8 rows, 768 x 50257            logits 15, join 4.8 us                     5.2 TB/s of weights
//   backward, 13107 rows, 768 x 50257       pack 42, G 968, dW 890, dx 1290, dx's end 12 us
//   (products alone by a library 910, 1097 and 970 us)
//   backward, 501 rows, 500 x 10007 fp16    pack 10, G 19, dW 20, dx 19, dx's end 8 us
#include "tiles.h"

#include "chunks.h"

namespace {

constexpr float kLog2E = 1.44269504f, kLn2 = 0.693147181f;

struct HeadState {          // device
  int32_t count;            // rows that count
  float factor, lift;       // G's factor besides dloss, and its logarithm to base 2
  float scale;              // what dx and dW are multiplied with in the end
};
struct HeadRow {            // a row that counts; logarithms to base 2
  float logit;              // its target's logit; forward: less the shift
  float lse, d;             // backward; forward, lse: the target's logit less the shift as its tile has it
  int32_t target, row;      // its place among all rows
};
// A row's shift, forward: its target's logit but for the low bits (a 32nd of it at most), which say the target, so that the
// wave that has it knows.  (All targets loaded in the end of every tile of 256 x 256: 16384 x 768 x 51200 1088 -> 1160 us.)
constexpr uint32_t kPlace = 0x3FFFF;
APEXW_DEV float with_place(float logit, int target) {
  return __uint_as_float((__float_as_uint(logit) & ~kPlace) | ((uint32_t)target & kPlace));
}
struct HeadArgs {
  const HeadState* state;
  HeadRow* rows;
  const float* shift;       // one a row, of the exponents of its tiles
  float* sums;              // [columns of a wave or tile][row]: log2 of the sum of 2^(l log2 e - shift), or few rows' pairs
  int64_t sums_ld;
};

// ---------------------------------------------------------------------------
// Rows that count, packed
// ---------------------------------------------------------------------------

struct PackArgs {
  const uint16_t *x, *w;
  const void* target;
  const float *lse, *dloss;   // backward
  uint16_t* packed;
  HeadState* state;
  HeadRow* rows;
  float* shift;
  float *loss, *lse_out;      // forward: zeros for the rows that do not count
  void* dx;                   // the same, backward
  int64_t n, x_stride, w_stride, dloss_stride, ignore;
  int32_t width, wide, vocab, id64, per, mean;
};

APEXW_DEV int64_t target_of(const PackArgs& a, int64_t i) {
  return a.id64 ? APEXW_GLOBAL(const int64_t, a.target)[i] : (int64_t)APEXW_GLOBAL(const int32_t, a.target)[i];
}
APEXW_DEV bool counts(const PackArgs& a, int64_t t) { return t != a.ignore && t >= 0 && t < a.vocab; }

template <class T, class F> APEXW_DEV T over_workgroup(T x, T* lds, F&& f) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) x = f(x, __shfl_xor(x, off, 64));
  if (lane_id() == 0) lds[threadIdx.x >> 6] = x;
  __syncthreads();
  x = f(f(lds[0], lds[1]), f(lds[2], lds[3]));
  __syncthreads();
  return x;
}

// A workgroup has `per` rows, 256 at a time; how many rows before them count it finds by itself.  A wave takes a row at
// a time: copies it, and forms its target's logit on the way.
template <int DT> __global__ __launch_bounds__(256) void head_pack_kernel(PackArgs a, Pad weights, int groups) {
  if ((int)blockIdx.x >= groups) {   // the weights, copied to whole chunks
    if (weights.rows * ((weights.width + 7) / 8) < (1ll << 31)) pad_rows<uint32_t>(weights, blockIdx.x - groups, gridDim.x - groups);
    else pad_rows<uint64_t>(weights, blockIdx.x - groups, gridDim.x - groups);
    return;
  }
  __shared__ int ints[4];
  __shared__ float floats[4];
  __shared__ int place[256];
  const int64_t first = (int64_t)blockIdx.x * a.per, end = first + a.per < a.n ? first + a.per : a.n;
  const bool last = (int)blockIdx.x == groups - 1;
  int before = 0;
  float most = 0.0f;
  const bool find_most = last && a.dloss;
  constexpr int U = 16;   // loads in flight
  for (int64_t i0 = threadIdx.x; i0 < first; i0 += 256 * U) {
    int64_t t[U];
#pragma unroll
    for (int u = 0; u < U; ++u) t[u] = i0 + 256 * u < first ? target_of(a, i0 + 256 * u) : -1;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool c = counts(a, t[u]);
      before += c;
      if (find_most && c) most = fmaxf(most, fabsf(a.dloss[(i0 + 256 * u) * a.dloss_stride]));
    }
  }
  before = over_workgroup(before, ints, [](int p, int q) { return p + q; });

  for (int64_t from = first; from == first || from < end; from += 256) {
    const int64_t to = from + 256 < end ? from + 256 : end;
    const int64_t mine = from + threadIdx.x;
    const bool has = mine < to && counts(a, target_of(a, mine));
    const uint64_t ballot = __ballot(has);
    if (lane_id() == 0) ints[threadIdx.x >> 6] = __builtin_popcountll(ballot);
    __syncthreads();
    int at = before + __builtin_popcountll(ballot & ((1ull << lane_id()) - 1ull));
    for (int w = 0; w < (int)(threadIdx.x >> 6); ++w) at += ints[w];
    const int all = before + ints[0] + ints[1] + ints[2] + ints[3];
    place[threadIdx.x] = has ? at : -1;
    __syncthreads();
    if (mine < to && !has) {
      if (a.loss) a.loss[mine] = 0.0f;
      if (a.lse_out) a.lse_out[mine] = 0.0f;
    }
    if (last && a.dloss && has) most = fmaxf(most, fabsf(a.dloss[mine * a.dloss_stride]));
    if (last && to == end) {
      if (a.dloss) most = over_workgroup(most, floats, [](float p, float q) { return fmaxf(p, q); });
      if (threadIdx.x == 0) {
        // The largest dloss is divided out of G and multiplied into the sums: a row that is far from its target then has
        // -2^14 there, which no rounding changes (where all rows have one dloss, its own rounding would be every row's).
        // The 2^14 leave fp16 its range below: a G of 2^-28 of the largest keeps its bits, one of 2^-39 is the least that is
        // not 0 (largest 1: 2^-14 and 2^-25, and a quarter of G was 0 where logits spread by 3 over 50257 words); 2^2 are
        // left above.
        const float mean = a.mean && all > 0 ? 1.0f / (float)all : 1.0f;
        const bool use = most >= 0x1p-100f && most < INFINITY;
        const float factor = use ? 0x1p14f / most : 1.0f, scale = use ? most * 0x1p-14f * mean : mean;
        *a.state = HeadState{all, factor, log2f(factor), scale};
      }
    }

    const int chunks = a.wide / 8, rows = (int)(to - from), lane = lane_id();
    for (int r = threadIdx.x >> 6; r < rows; r += 4) {
      const int64_t i = from + r;
      const int p = uniform(place[r]);
      if (p < 0) {
        if (!a.dx) continue;
        uint16_t* dx = (uint16_t*)a.dx + i * a.width;
        for (int c = lane; c < chunks; c += 64) {
          const int n = clamp8(a.width - c * 8);
          if (n == 8) APEXW_GLOBAL(Chunk, dx + c * 8)->v = u32x4{0u, 0u, 0u, 0u};
          else for (int j = 0; j < n; ++j) APEXW_GLOBAL(uint16_t, dx)[c * 8 + j] = 0;
        }
        continue;
      }
      const int target = (int)target_of(a, i);
      const uint16_t *x = a.x + i * a.x_stride, *w = a.w + target * a.w_stride;
      float dot = 0.0f;
#pragma unroll 4
      for (int c = lane; c < chunks; c += 64) {
        const int n = clamp8(a.width - c * 8);
        const u32x4 xv = load_chunk(x + c * 8, n), wv = load_chunk(w + c * 8, n);
        *(u32x4*)&a.packed[(int64_t)p * a.wide + c * 8] = xv;
        float xs[8], ws[8];
        values<DT>(xv, xs), values<DT>(wv, ws);
#pragma unroll
        for (int j = 0; j < 8; ++j) dot = fmaf(xs[j], ws[j], dot);
      }
      dot = wave_sum(dot);
      if (lane) continue;
      HeadRow row{dot * kLog2E, 0.0f, 0.0f, target, (int32_t)i};
      float shift = row.logit - row.logit == 0.0f ? row.logit : 0.0f;
      if (a.lse) {
        row.lse = a.lse[i] * kLog2E, row.d = a.dloss[i * a.dloss_stride];
        const uint32_t bits = __float_as_uint(log2f(fabsf(row.d)) - row.lse);
        shift = __uint_as_float((bits & ~1u) | (row.d < 0.0f));
      } else {
        shift = with_place(shift, target);
        row.logit = fmaf(dot, kLog2E, -shift);
      }
      a.rows[p] = row, a.shift[p] = shift;
    }
    before = all;
  }
}

// ---------------------------------------------------------------------------
// Tiles of logits
// ---------------------------------------------------------------------------

// A tile's first row and column, which `locate` packs into one number
APEXW_DEV int64_t tile_at(int64_t row, int64_t col) { return row << 32 | col; }

template <int FA, int FB, class Acc> APEXW_DEV void mask_columns(Acc& acc, int wn, int cols, float to) {
  const int c0 = 4 * (lane_id() >> 4);
#pragma unroll
  for (int j = 0; j < FB; ++j)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const bool out = wn + 16 * j + c0 + q >= cols;
#pragma unroll
      for (int i = 0; i < FA; ++i) acc[i][j][q] = out ? to : acc[i][j][q];
    }
}

// Each row's shift
template <int FA> struct Shifts {
  float v[FA];
  __device__ __forceinline__ void load(const float* shift, int64_t row0, int row, int rows) {
#pragma unroll
    for (int i = 0; i < FA; ++i) v[i] = shift[row0 + min(row + 16 * i, rows - 1)];
  }
  __device__ __forceinline__ void arrived() {
#pragma unroll
    for (int i = 0; i < FA; ++i) asm volatile("" : "+v"(v[i]));
  }
};

// Forward: each row's sum of exponentials over a wave's columns, relative to its shift.  That is a maximum's part as long as no
// logit is 83 above it (2^120) and one is 83 below or more; the rows of a block where this is not so are summed again from
// their maximum.  The packing's target's logit is off from the tile's by their orders of summing (3e-4 at logits of
// 1000), so the wave that has the target leaves its exponent as it is in the sum, where the join puts the packing's for it
// (which is the nearer one): a row certain of its target has a loss of 0, not of that difference.
// (16384 x 768 x 51200 1094 -> 1107 us, 8192 x 4096 x 128256 6266 -> 6313.)
struct Sums {
  HeadArgs h;
  template <int FA> using Rows = Shifts<FA>;
  template <class R> __device__ __forceinline__ void load(R& known, int64_t out0, int row, int rows) const {
    known.load(h.shift, out0 >> 32, row, rows);
  }
  template <class S> static constexpr int stores() { return 0; }
  template <class S, int kWM, class Acc, class R>
  __device__ __forceinline__ void write(const ExpertArgs& g, Acc& acc, const R& known, uint16_t* lds, int down, int across,
                                        int rows, int cols, int64_t out0) const {
    constexpr int FA = kWM / 16, FB = S::WN / 16;
    const int wm = down * kWM, wn = across * S::WN, lane = lane_id();
    const int64_t row0 = out0 >> 32;
    const int col0 = (int)(uint32_t)out0;
    // tiles of one wave's rows: the waves' sums are joined here, since what few rows take is the last launch's time
    constexpr bool kJoin = S::BM == S::WM;
    constexpr int kAcross = S::BN / S::WN;
    if (!kJoin && wn >= cols) return;
    if (wn + S::WN > cols) mask_columns<FA, FB>(acc, wn, cols, -INFINITY);
    float* parts = (float*)(lds + S::kStages * S::kStageElems);
    float* to = kJoin ? parts + across * S::WM : h.sums + (col0 + wn) / S::WN * h.sums_ld + row0 + wm;
    const uint32_t place = (uint32_t)(col0 + wn) & kPlace;
#pragma unroll
    for (int i = 0; i < FA; ++i) {
      const float shift = known.v[i];
      float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int j = 0; j < FB; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) s[q] += __builtin_amdgcn_exp2f(fmaf(acc[i][j][q], kLog2E, -shift));
      float sum = (s[0] + s[1]) + (s[2] + s[3]);
      sum += __shfl_xor(sum, 16, 64);
      sum += __shfl_xor(sum, 32, 64);
      float part = __builtin_amdgcn_logf(sum);   // to base 2
      if (__builtin_expect(__ballot(!(fabsf(part) < 120.0f)) != 0, 0)) {
        float m = acc[i][0][0];
#pragma unroll
        for (int j = 0; j < FB; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) m = fmaxf(m, acc[i][j][q]);
        m = fmaxf(m, __shfl_xor(m, 16, 64));
        m = fmaxf(m, __shfl_xor(m, 32, 64));
        const float top = m == -INFINITY ? 0.0f : m;
        sum = 0.0f;
#pragma unroll
        for (int j = 0; j < FB; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) sum += __builtin_amdgcn_exp2f((acc[i][j][q] - top) * kLog2E);
        sum += __shfl_xor(sum, 16, 64);
        sum += __shfl_xor(sum, 32, 64);
        part = fmaf(top, kLog2E, -shift) + __builtin_amdgcn_logf(sum);
      }
      if (lane < 16 && wm + 16 * i + lane < rows) to[16 * i + lane] = part;
      uint32_t t = (__float_as_uint(shift) & kPlace) - place;
      if (__builtin_expect(__ballot(t < S::WN) != 0, 0)) {
        const int r = wm + 16 * i + (lane & 15);
        if (g.n > (int)kPlace) t = (uint32_t)(h.rows[row0 + min(r, rows - 1)].target - col0 - wn);
        float logit = 0.0f;
#pragma unroll
        for (int j = 0; j < FB; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) logit = (t & ~12u) == 16u * j + q ? acc[i][j][q] : logit;
        if (t < S::WN && r < rows && (int)(t >> 2 & 3u) == lane >> 4) h.rows[row0 + r].lse = fmaf(logit, kLog2E, -shift);
      }
    }
    if constexpr (kJoin) {
      barrier();
      const int r = threadIdx.x;
      if (r < rows && r < kWM) {
        float top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kAcross; ++w) top = fmaxf(top, parts[w * S::WM + r]);
        const float from = top == -INFINITY ? 0.0f : top;
#pragma unroll
        for (int w = 0; w < kAcross; ++w) sum += __builtin_amdgcn_exp2f(parts[w * S::WM + r] - from);
        h.sums[col0 / S::BN * h.sums_ld + row0 + r] = from + __builtin_amdgcn_logf(sum);
      }
    }
  }
};

// y 2^(x unit) more, as a sum from the larger x
APEXW_DEV void add_sum(float2& a, float2 b, float unit) {
  const float top = fmaxf(a.x, b.x), to = top == -INFINITY ? 0.0f : top;
  a = make_float2(top, a.y * __builtin_amdgcn_exp2f((a.x - to) * unit) + b.y * __builtin_amdgcn_exp2f((b.x - to) * unit));
}

// Forward of few rows, up to one tile's, as they stand: without a packing launch before it a tile leaves its maximum and
// the sum from it (one logarithm of both would round at the logits' size), and the tile that has a row's target leaves its
// logit.  (8 rows, 768 x 50257: 20.2 us a call, 26.7 with the
// packing, 5.6 of it its launch.)
struct FewTargets {
  const uint32_t* id;
  int64_t ignore;
  int32_t id64, vocab;
  // (loaded in words, so that nothing waits for them before the end)
  __device__ __forceinline__ uint32_t low(int row) const { return APEXW_GLOBAL(const uint32_t, id)[id64 ? 2 * row : row]; }
  __device__ __forceinline__ uint32_t high(int row) const { return APEXW_GLOBAL(const uint32_t, id)[id64 ? 2 * row + 1 : row]; }
  __device__ __forceinline__ int target(uint32_t lo, uint32_t hi) const {   // -1 for a row that does not count
    const int64_t t = id64 ? (int64_t)((uint64_t)hi << 32 | lo) : (int64_t)(int32_t)lo;
    return t != ignore && t >= 0 && t < vocab ? (int)t : -1;
  }
};
struct FewSums {
  HeadArgs h;
  FewTargets targets;
  float* logits;   // of each row's target
  template <int FA> struct Rows {
    uint32_t lo[FA], hi[FA];
    __device__ __forceinline__ void arrived() {
#pragma unroll
      for (int i = 0; i < FA; ++i) asm volatile("" : "+v"(lo[i]), "+v"(hi[i]));
    }
  };
  template <int FA> __device__ __forceinline__ void load(Rows<FA>& known, int64_t, int row, int rows) const {
#pragma unroll
    for (int i = 0; i < FA; ++i) {
      const int r = min(row + 16 * i, rows - 1);
      known.lo[i] = targets.low(r), known.hi[i] = targets.high(r);
    }
  }
  template <class S> static constexpr int stores() { return 0; }
  template <class S, int kWM, class Acc, class R>
  __device__ __forceinline__ void write(const ExpertArgs& g, Acc& acc, const R& known, uint16_t* lds, int down, int across,
                                        int rows, int cols, int64_t out0) const {
    constexpr int FA = kWM / 16, FB = S::WN / 16, kAcross = S::BN / S::WN;
    static_assert(S::BM == S::WM, "a wave has a tile's rows");
    const int wn = across * S::WN, lane = lane_id(), col0 = (int)(uint32_t)out0;
    float2* parts = (float2*)(lds + S::kStages * S::kStageElems);
    if (wn + S::WN > cols) mask_columns<FA, FB>(acc, wn, cols, -INFINITY);
#pragma unroll
    for (int i = 0; i < FA; ++i) {
      const int r = 16 * i + (lane & 15), t = r < rows ? targets.target(known.lo[i], known.hi[i]) - col0 - wn : -1;
      if (__ballot(t >= 0 && t < S::WN)) {
#pragma unroll
        for (int j = 0; j < FB; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (t == 16 * j + 4 * (lane >> 4) + q) logits[r] = acc[i][j][q];
      }
      float m = acc[i][0][0];
#pragma unroll
      for (int j = 0; j < FB; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) m = fmaxf(m, acc[i][j][q]);
      m = fmaxf(m, __shfl_xor(m, 16, 64));
      m = fmaxf(m, __shfl_xor(m, 32, 64));
      const float top = m == -INFINITY ? 0.0f : m;
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < FB; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) sum += __builtin_amdgcn_exp2f((acc[i][j][q] - top) * kLog2E);
      sum += __shfl_xor(sum, 16, 64);
      sum += __shfl_xor(sum, 32, 64);
      if (lane < 16) parts[across * S::WM + 16 * i + lane] = make_float2(m, sum);
    }
    barrier();
    const int r = threadIdx.x;
    if (r >= rows || r >= kWM) return;
    float2 all = parts[r];
#pragma unroll
    for (int w = 1; w < kAcross; ++w) add_sum(all, parts[w * S::WM + r], kLog2E);
    ((float2*)h.sums)[col0 / S::BN * h.sums_ld + r] = all;
  }
};
// One tile's rows against all columns
struct FewJobs {
  int rows, tiles;
  __device__ __forceinline__ Job get(int i) const {
    const int64_t t = (int64_t)i * gridDim.x + blockIdx.x;
    return t < tiles ? Job{0, 0, rows, 0, (int)t, 0} : Job{-1, 0, 0, 0, 0, 0};
  }
};
template <int DT> __global__ __launch_bounds__(Small::kThreads, 2) void head_few_kernel(ExpertArgs g, FewSums out, HeadState* state) {
  __shared__ __attribute__((aligned(16))) uint16_t lds[Small::kLds];
  FewJobs jobs{(int)g.rows, (g.n + Small::BN - 1) / Small::BN};
  stream<Small, false, false, DT, true>(g, jobs, [&](const Job& j, Span& a, Span& b, int& rows, int& cols, int64_t& out0) {
    const int64_t col = j.col * Small::BN;
    rows = j.last, cols = g.n - (int)col, out0 = tile_at(0, col);
    a.template set<false>(g.a, g.lda, rows, g.wide, Small::BM);
    b.template set<false>(g.b + col * g.ldb, g.ldb, cols, g.wide, Small::BN);
  }, out, lds);
  if (blockIdx.x || threadIdx.x >= 64) return;
  const int r = (int)threadIdx.x < g.rows ? threadIdx.x : 0;
  const uint64_t count = __ballot((int)threadIdx.x < g.rows && out.targets.target(out.targets.low(r), out.targets.high(r)) >= 0);
  if (threadIdx.x == 0) state->count = __builtin_popcountll(count);
}

// Backward: the tile's part of G, whole chunks of columns; a tile of 256 x 256, whose registers are all in use, leaves
// the targets' elements to a launch behind it
constexpr bool targets_apart(int shape) { return shape == 3; }
template <int DT> struct Prob {
  HeadArgs h;
  int32_t first;   // the piece's first column
  template <int FA> using Rows = Shifts<FA>;
  template <class R> __device__ __forceinline__ void load(R& known, int64_t out0, int row, int rows) const {
    known.load(h.shift, out0 >> 32, row, rows);
  }
  template <class S> static constexpr int stores() { return Store<DT>::template stores<S>(); }
  template <class S, int kWM, class Acc, class R>
  __device__ __forceinline__ void write(const ExpertArgs& g, Acc& acc, const R& known, uint16_t* lds, int down, int across,
                                        int rows, int cols, int64_t out0) const {
    constexpr int FA = kWM / 16, FB = S::WN / 16;
    const float lift = h.state->lift;
#pragma unroll
    for (int i = 0; i < FA; ++i) {
      const uint32_t bits = __float_as_uint(known.v[i]);
      const float shift = __uint_as_float(bits & ~1u) + lift;
#pragma unroll
      for (int j = 0; j < FB; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) acc[i][j][q] = __builtin_amdgcn_exp2f(fmaf(acc[i][j][q], kLog2E, shift));
      if (__ballot(bits & 1u)) {
#pragma unroll
        for (int j = 0; j < FB; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) acc[i][j][q] = bits & 1u ? -acc[i][j][q] : acc[i][j][q];
      }
      if constexpr (!std::is_same_v<S, Large>) {
        const int r = down * kWM + 16 * i + (lane_id() & 15);
        const HeadRow& row = h.rows[(out0 >> 32) + min(r, rows - 1)];
        const int t = row.target - first - (int)(uint32_t)out0 - across * S::WN;
        if (__ballot(t >= 0 && t < S::WN)) {
          const float d = row.d * h.state->factor;
#pragma unroll
          for (int j = 0; j < FB; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) acc[i][j][q] -= t == 16 * j + 4 * (lane_id() >> 4) + q ? d : 0.0f;
        }
      }
    }
    if (cols < S::BN) mask_columns<FA, FB>(acc, across * S::WN, cols, 0.0f);
    Store<DT>::template put<S, kWM>(g, acc, lds, down, across, rows, (cols + 7) / 8 * 8,
                                    (out0 >> 32) * g.ldo + (int64_t)(uint32_t)out0, Same{});
  }
};

// The targets' elements of the piece's G, from the logits that the packing formed
template <int DT> __global__ __launch_bounds__(256) void head_targets_kernel(HeadArgs h, int first, int cols, void* g, int64_t ldg) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= h.state->count) return;
  const HeadRow row = h.rows[i];
  const int t = row.target - first;
  if (t >= 0 && t < cols) store_elem<DT>(g, i * ldg + t, (exp2f(row.logit - row.lse) - 1.0f) * row.d * h.state->factor);
}

template <class S, int DT, class Out> __global__ __launch_bounds__(S::kThreads, 2) void head_logits_kernel(ExpertArgs g, Out out) {
  __shared__ __attribute__((aligned(16))) uint16_t lds[S::kLds];
  RowJobs<true> jobs(g, S::BM, S::BN);
  stream<S, false, false, DT, true>(g, jobs, [&](const Job& j, Span& a, Span& b, int& rows, int& cols, int64_t& out0) {
    const int64_t row = j.first + j.row, col = j.col * S::BN;
    rows = j.last - (int)row, cols = g.n - (int)col, out0 = tile_at(row, col);
    a.template set<false>(g.a + row * g.lda, g.lda, rows, g.wide, S::BM);
    b.template set<false>(g.b + col * g.ldb, g.ldb, cols, g.wide, S::BN);
  }, out, lds);
}

// ---------------------------------------------------------------------------
// The rows' statistics joined, and their mean
// ---------------------------------------------------------------------------

// 16 rows a workgroup, a 64th of the sums a thread; `few` rows as they stand, or 0
__global__ __launch_bounds__(1024) void head_join_kernel(HeadArgs h, int parts, int few, FewTargets targets, float* __restrict__ loss,
                                                         float* __restrict__ lse) {
  __shared__ float2 lds[16][16];
  const int r = threadIdx.x & 15, q = threadIdx.x >> 4;
  const int64_t first = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 16, row = first + r;
  const int count = few ? few : h.state->count;
  if (first >= count) return;
  float2 all = {-INFINITY, 0.0f};
  const float unit = few ? kLog2E : 1.0f;
  if (row < count) {
    if (few) {
#pragma unroll 8
      for (int t = q; t < parts; t += 64) add_sum(all, ((const float2*)h.sums)[t * h.sums_ld + row], unit);
    } else {
#pragma unroll 8
      for (int t = q; t < parts; t += 64) add_sum(all, make_float2(h.sums[t * h.sums_ld + row], 1.0f), unit);
    }
  }
  for (int off = 16; off < 64; off <<= 1) add_sum(all, make_float2(__shfl_xor(all.x, off, 64), __shfl_xor(all.y, off, 64)), unit);
  if ((q & 3) == 0) lds[q >> 2][r] = all;
  __syncthreads();
  if (q != 0 || row >= count) return;
#pragma unroll
  for (int i = 1; i < 16; ++i) add_sum(all, lds[i][r], unit);
  const float top = all.x == -INFINITY ? 0.0f : all.x, shift = h.shift[row];
  if (few) {
    const bool has = targets.target(targets.low((int)row), targets.high((int)row)) >= 0;
    const float sum = log2f(all.y) * kLn2;
    lse[row] = has ? top + sum : 0.0f;
    loss[row] = has ? (top - shift) + sum : 0.0f;
    return;
  }
  const HeadRow& info = h.rows[row];
  const float others = all.y - __builtin_amdgcn_exp2f(info.lse - top);
  all = others <= 0.0f ? make_float2(-INFINITY, 0.0f) : make_float2(top, others);
  add_sum(all, make_float2(info.logit, 1.0f), 1.0f);
  const float sum = all.x + log2f(all.y);
  lse[info.row] = (shift + sum) * kLn2;
  const float above = (sum - info.logit) * kLn2;   // (not below 0 but for roundings; NaN stays)
  loss[info.row] = above < 0.0f ? 0.0f : above;
}

// The sum of the rows' losses, or their mean over the rows that count
__global__ __launch_bounds__(1024) void head_total_kernel(const HeadState* state, const float* loss, int64_t n, int mean, float* total) {
  __shared__ double parts[16];
  double s = 0.0;
#pragma unroll 4
  for (int64_t i = threadIdx.x; i < n; i += 1024) s += (double)loss[i];
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
  if (lane_id() == 0) parts[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x) return;
  s = 0.0;
  for (int i = 0; i < 16; ++i) s += parts[i];
  *total = (float)(mean ? s / (double)state->count : s);
}

// ---------------------------------------------------------------------------
// The two products with G
// ---------------------------------------------------------------------------

template <int OD> struct Scaled {
  const HeadState* state;
  template <int FA> using Rows = NoRows;
  template <class R> __device__ __forceinline__ void load(R&, int64_t, int, int) const {}
  template <class S> static constexpr int stores() { return Store<OD>::template stores<S>(); }
  template <class S, int kWM, class Acc>
  __device__ __forceinline__ void write(const ExpertArgs& g, Acc& acc, const NoRows&, uint16_t* lds, int down, int across,
                                        int rows, int cols, int64_t out0) const {
    const float scale = state->scale;
    Store<OD>::template put<S, kWM>(g, acc, lds, down, across, rows, cols, out0, [scale](f32x4 v, int, int) {
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] *= scale;
      return v;
    });
  }
};

// dW of the piece: [columns of G] x [width of x], over the rows that count
template <class S, int DT, int OD, class Out>
__global__ __launch_bounds__(S::kThreads, 2) void head_weight_kernel(ExpertArgs g, Out out) {
  __shared__ __attribute__((aligned(16))) uint16_t lds[S::kLds];
  if (g.splits == 1) zero_weights<OD>(g);
  WeightJobs jobs(g, S::BM, S::BN);
  stream<S, true, true, DT, false>(g, jobs, [&](const Job& j, Span& a, Span& b, int& rows, int& cols, int64_t& out0) {
    const int64_t row = j.row, col = j.col * S::BN, first = j.first;
    rows = g.n - (int)row, cols = g.k - (int)col;
    out0 = j.split * g.split_stride + row * g.k + col;
    a.template set<true>(g.a + first * g.lda + row, g.lda, (rows + 7) / 8 * 8, j.last - j.first, S::BM);
    b.template set<true>(g.b + first * g.ldb + col, g.ldb, (cols + 7) / 8 * 8, j.last - j.first, S::BN);
  }, out, lds);
}
template <int OD>
__global__ __launch_bounds__(256) void head_join_weight_kernel(ExpertArgs g, const HeadState* state, const float* __restrict__ partial) {
  const int rows = state->count, len = rows ? split_rows(rows, g.splits) : 1, parts = (rows + len - 1) / len;
  const int64_t n = (int64_t)g.n * g.k;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256)
    store_elem<OD>(g.out, i, join(partial + i, g.split_stride, parts) * state->scale);
}

// The piece's part of dx: in fp32, added to the pieces before (sums of their own, added up in the end, are as fast: 100000
// rows, 1024 x 30010, dx alone 12.4 ms added, 12.5 apart; 16384, 768 x 50257 2.84 and 2.83)
template <class S, int DT, bool kAdd> __global__ __launch_bounds__(S::kThreads, 2) void head_rows_kernel(ExpertArgs g) {
  __shared__ __attribute__((aligned(16))) uint16_t lds[S::kLds];
  RowJobs<true> jobs(g, S::BM, S::BN);
  stream<S, false, true, DT, true>(g, jobs, [&](const Job& j, Span& a, Span& b, int& rows, int& cols, int64_t& out0) {
    const int64_t row = j.first + j.row, col = j.col * S::BN;
    const int k0 = j.split * g.part, wide = g.wide - k0 < g.part ? g.wide - k0 : g.part;
    const int deep = g.k - k0 < g.part ? g.k - k0 : g.part;
    rows = j.last - (int)row, cols = g.n - (int)col, out0 = j.split * g.split_stride + row * g.ldo + col;
    a.template set<false>(g.a + row * g.lda + k0, g.lda, rows, wide, S::BM);
    b.template set<true>(g.b + k0 * g.ldb + col, g.ldb, (cols + 7) / 8 * 8, deep, S::BN);
  }, Store<APEXW_F32, kAdd>(), lds);
}

// dx: the parts' sums, scaled, each row at its place
template <int DT> __global__ __launch_bounds__(256) void head_dx_kernel(HeadArgs h, const float* __restrict__ sums, int64_t stride,
                                                                       int splits, int width, uint16_t* dx) {
  const int count = h.state->count, per = (width + 7) / 8;
  const float scale = h.state->scale;
  const int64_t n = (int64_t)count * per;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / per;
    const int c = (int)(i - r * per) * 8, has = clamp8(width - c);
    const float* p = sums + r * width + c;
    uint16_t* to = dx + (int64_t)h.rows[r].row * width + c;
    if (has == 8) {
      float v[8] = {};
#pragma unroll 4
      for (int s = 0; s < splits; ++s) {
        const u32x4 lo = APEXW_GLOBAL(const Chunk32, p + s * stride)->v, hi = APEXW_GLOBAL(const Chunk32, p + s * stride + 4)->v;
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] += __uint_as_float(lo[q]), v[4 + q] += __uint_as_float(hi[q]);
      }
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] *= scale;
      APEXW_GLOBAL(Chunk, to)->v = rounded<DT>(v);
    } else {
      for (int q = 0; q < has; ++q) {
        float v = 0.0f;
        for (int s = 0; s < splits; ++s) v += p[s * stride + q];
        store_elem<DT>(to, q, v * scale);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------

int64_t whole(int64_t bytes) { return (bytes + 255) / 256 * 256; }

// The time of a product whose tiles the chip takes in rounds, in us: a stage's when every workgroup is at work and with
// few, the end of a tile that is written in 16 bits or in fp32 (a round's 64 MB at once), and the launch and bytes of
// parts that are joined.  whole_rounds: a last round takes as long as the others; else its tiles are cut.  The rates
// are those of dx of 16384, 13107 (156 tiles of 256 x 256: whole 579 us, in three parts 457, in four 518), 2048, 500 and
// 64 rows with 768 x 21760, 1024 x 32000, 504 x 10007 and 768 x 50257, each shape in 1 to 16 parts.
struct Rate {
  float most, least, end16, end32;
  int slots, bm, bn;
};
template <class S> Rate rate(float most, float least, float end16, float end32) {
  return {most, least, end16, end32, apexw_cu_count() * S::kPerCU, S::BM, S::BN};
}
Rate rate_of(int shape) {
  if (shape == 3) return rate<Large>(1.65f, 1.35f, 9.0f, 30.0f);
  if (shape == 2) return rate<Wide>(1.13f, 0.85f, 5.0f, 9.0f);
  if (shape == 1) return rate<Mid>(0.72f, 0.48f, 4.0f, 7.0f);
  return rate<Small>(0.6f, 0.42f, 3.0f, 4.0f);
}
float time_of(int shape, int64_t down, int64_t across, int64_t depth, int splits, bool whole_rounds, bool fp32, float join_bytes) {
  const Rate r = rate_of(shape);
  const float tiles = (float)((down + r.bm - 1) / r.bm) * (float)((across + r.bn - 1) / r.bn);
  const float rounds = tiles * (float)splits / (float)r.slots, full = floorf(rounds), rest = rounds - full;
  const float stages = ceilf((float)((depth + kDepth - 1) / kDepth) / (float)splits), end = fp32 ? r.end32 : r.end16;
  const float join = splits > 1 ? 5.0f + (float)(splits - 1) * join_bytes / 4e6f : 0.0f;
  if (rounds <= 1.0f) return stages * (r.least + (r.most - r.least) * rounds) + 3.0f + (end - 3.0f) * rounds + join;
  const float last = rest == 0.0f ? 0.0f : whole_rounds || splits > 1 || rest > 0.5f ? 1.0f : rest > 0.25f ? 0.6f : 0.4f;
  return (full + last) * (stages * r.most + end) + join;
}
// the shape and parts of the least time; parts have to gain a tenth
Cut best_cut(int least_shape, int64_t down, int64_t across, int64_t depth, bool may_split, bool whole_rounds, bool fp32,
             float join_bytes) {
  Cut best{0, 0, 0.0f};
  for (int shape = least_shape; shape < 4; ++shape)
    for (int splits = 1; splits == 1 || (may_split && splits <= 64 && splits * 4 * kDepth <= depth); ++splits) {
      if (splits > 4 && (splits & (splits - 1))) continue;
      const float t = time_of(shape, down, across, depth, splits, whole_rounds, fp32 || splits > 1, join_bytes);
      const float cost = splits > 1 ? 1.1f * t : t;
      if (best.splits == 0 || cost < best.cost) best = {shape, splits, cost};
    }
  return best;
}

// Bytes of G that a piece may have.  (Between 128 MB and 4 GB the time changes by what the pieces' tiles leave of the
// chip's rounds alone: 8192 x 4096 x 128256 19.9 to 20.6 ms.)
constexpr int64_t kPiece = 1ll << 30;
// The products of a piece of `cols` columns of the vocabulary
struct Piece {
  int64_t cols;
  Cut logits, dw, dx;
  float cost;
  Piece() = default;
  Piece(int64_t c, int64_t n, int64_t width, bool need_dx, bool need_dw) : cols(c) {
    logits = best_cut(0, n, cols, width, false, false, false, 0.0f);
    if (targets_apart(logits.shape)) {   // a launch more
      const float other = time_of(2, n, cols, width, 1, false, false, 0.0f);
      if (other < logits.cost + 4.0f) logits = {2, 1, other};
      else logits.cost += 4.0f;
    }
    dw = best_cut(2, cols, width, n, true, true, false, 8.0f * (float)cols * (float)width);
    dx = best_cut(0, n, width, cols, true, false, true, 8.0f * (float)n * (float)width);
    // (sums of dx that are written and read again)
    cost = logits.cost + (need_dw ? dw.cost : 0.0f) + (need_dx ? dx.cost + 8.0f * (float)n * (float)width / 4e6f : 0.0f);
  }
};

// (Shapes, parts and pieces are those of all n rows: how many count is known on the device alone.  Rows that do not count
// make no tiles, but a batch that is mostly masked runs in tiles chosen for the whole of it.)
struct HeadPlan {
  int64_t n, width, wide, vocab, w_stride;
  bool copy_w;
  int64_t at_rows, at_shift, at_x, at_w, at_parts, at_g, at_sums, at_dw, bytes;
  int64_t parts_ld, piece_ld;
  Cut cut;                 // forward
  Piece piece, last;       // backward
  HeadPlan(const void* w, int64_t stride, int64_t n_, int64_t width_, int64_t vocab_, bool backward, bool need_dx, bool need_dw)
      : n(n_), width(width_), wide((width_ + 7) / 8 * 8), vocab(vocab_), w_stride(stride) {
    copy_w = !k_rows_ok(w, stride, width);
    if (copy_w) w_stride = wide;
    at_rows = 256;
    at_shift = at_rows + whole(n * (int64_t)sizeof(HeadRow));
    at_x = at_shift + whole(n * 4);
    at_w = at_x + whole(n * wide * 2);
    int64_t at = at_w + (copy_w ? whole(vocab * wide * 2) : 0);
    if (!backward) {
      cut = best_cut(0, n, vocab, width, false, false, false, 0.0f);
      parts_ld = (n + 15) / 16 * 16;
      at_parts = at, at += whole(parts_ld * parts() * (n <= Small::BM ? 8 : 4));   // (few rows: maximum and sum)
      bytes = at;
      return;
    }
    cut_pieces(need_dx, need_dw);
    piece_ld = (piece.cols + 7) / 8 * 8;
    at_g = at, at += whole(n * piece_ld * 2);
    at_sums = at, at += need_dx ? whole(dx(piece).splits * n * width * 4) : 0;
    int64_t parts = 0;
    if (need_dw)
      for (const Piece* q : {&piece, &last})
        if (q->dw.splits > 1 && q->dw.splits * q->cols > parts) parts = q->dw.splits * q->cols;
    at_dw = at, at += whole(parts * width * 4);
    bytes = at;
  }
  // Pieces of as many columns as G's bytes allow, or fewer, so that the tiles of their weights' gradient fill whole
  // rounds of the chip; the last piece has what is left
  void cut_pieces(bool need_dx, bool need_dw) {
    int64_t most = kPiece / (2 * (n > 0 ? n : 1)) / 256 * 256;
    most = most < 1024 ? 1024 : most;
    if (most >= vocab) {
      piece = last = Piece(vocab, n, width, need_dx, need_dw);
      return;
    }
    const int64_t across = (width + 255) / 256;
    float least = 0.0f;
    for (int i = 0; i < 5; ++i) {
      const int64_t cols = i == 0 ? most : apexw_cu_count() * i / across * 256;
      if (cols <= 0 || cols > most || 4 * cols < most) continue;
      const Piece p(cols, n, width, need_dx, need_dw);
      const int64_t count = (vocab - 1) / cols;
      Piece q(vocab - count * cols, n, width, need_dx, need_dw);
      const float cost = (float)count * p.cost + q.cost;
      if (least == 0.0f || cost < least) least = cost, piece = p, last = q;
    }
    last.dx = piece.dx;   // (the first piece writes every part's sums, to which the others add)
  }
  const Piece& at_column(int64_t v) const { return v + piece.cols <= vocab ? piece : last; }

  ExpertArgs args(int64_t columns) const {
    ExpertArgs g{};
    g.rows = n, g.experts = 1, g.splits = 1, g.part = INT32_MAX, g.n = (int32_t)columns, g.k = (int32_t)width;
    g.wide = (int32_t)wide, g.lda = wide, g.ldb = w_stride;
    return g;
  }
  ExpertArgs logits(const Piece& q) const {
    ExpertArgs g = args(q.cols);
    g.ldo = piece_ld;
    return g;
  }
  ExpertArgs dw(const Piece& q) const {
    ExpertArgs g = args(q.cols);
    g.lda = piece_ld, g.ldb = wide, g.ldo = width, g.split_stride = q.cols * width, g.splits = q.dw.splits;
    return g;
  }
  ExpertArgs dx(const Piece& q) const {
    ExpertArgs g = args(width);
    g.k = (int32_t)q.cols, g.wide = (int32_t)((q.cols + 7) / 8 * 8), g.lda = piece_ld, g.ldo = width, g.split_stride = n * width;
    cut_up(g, q.dx.splits, kDepth);
    return g;
  }
  int64_t parts() const {   // sums of a row
    const int64_t wave = cut.shape == 0 ? Small::BN : Large::WN;
    return (vocab + wave - 1) / wave;
  }
};
static_assert(Large::WN == 64 && Wide::WN == 64 && Mid::WN == 64 && Small::BM == Small::WM, "columns of a sum");

bool head_ok(int64_t n, int64_t width, int64_t vocab) {
  return n >= 0 && n <= INT32_MAX - 65536 && width > 0 && width <= kMostLd && vocab > 0 && vocab <= INT32_MAX - 65536;
}
// The join's workgroups along a grid's first dimension, which times 1024 threads has to stay below 2^32
constexpr int64_t kJoins = 1 << 21;
bool head_fits(const HeadPlan& p) { return p.n < 1ll << 26 && rows_tiles<Small>(p.args(p.vocab)) <= INT32_MAX; }

template <class S, int DT, class Out> void launch_logits_shape(const ExpertArgs& g, const Out& out, hipStream_t s) {
  hipLaunchKernelGGL((head_logits_kernel<S, DT, Out>), dim3(stream_grid<S>(rows_tiles<S>(g))), dim3(S::kThreads), 0, s, g, out);
}
template <int DT, class Out> void launch_logits(ExpertArgs g, int shape, const Out& out, hipStream_t s) {
  if (shape == 3) {
    launch_logits_shape<Large, DT>(g, out, s);
  } else if (shape == 2) {
    launch_logits_shape<Wide, DT>(g, out, s);
  } else if (shape == 1) {
    launch_logits_shape<Mid, DT>(g, out, s);
  } else {
    launch_logits_shape<Small, DT>(g, out, s);
  }
}
template <class S, int DT> void launch_dx_shape(const ExpertArgs& g, bool add, hipStream_t s) {
  const dim3 grid(stream_grid<S>(rows_tiles<S>(g) * g.splits)), block(S::kThreads);
  if (add) hipLaunchKernelGGL((head_rows_kernel<S, DT, true>), grid, block, 0, s, g);
  else hipLaunchKernelGGL((head_rows_kernel<S, DT, false>), grid, block, 0, s, g);
}
template <int DT> void launch_dx(ExpertArgs g, int shape, bool add, hipStream_t s) {
  if (shape == 3) {
    launch_dx_shape<Large, DT>(g, add, s);
  } else if (shape == 2) {
    launch_dx_shape<Wide, DT>(g, add, s);
  } else if (shape == 1) {
    launch_dx_shape<Mid, DT>(g, add, s);
  } else {
    launch_dx_shape<Small, DT>(g, add, s);
  }
}
template <int DT, int OD, class Out> void launch_dw_to(const ExpertArgs& g, int shape, const Out& out, hipStream_t s) {
  if (shape == 3)
    hipLaunchKernelGGL((head_weight_kernel<Large, DT, OD, Out>), dim3(stream_grid<Large>(weight_tiles<Large>(g) * g.splits)),
                       dim3(Large::kThreads), 0, s, g, out);
  else
    hipLaunchKernelGGL((head_weight_kernel<Wide, DT, OD, Out>), dim3(stream_grid<Wide>(weight_tiles<Wide>(g) * g.splits)),
                       dim3(Wide::kThreads), 0, s, g, out);
}
template <int DT> void launch_dw(const ExpertArgs& g, int shape, const HeadState* state, float* partial, hipStream_t s) {
  if (g.splits == 1) return launch_dw_to<DT, DT>(g, shape, Scaled<DT>{state}, s);
  ExpertArgs h = g;
  h.out = partial;
  launch_dw_to<DT, APEXW_F32>(h, shape, Store<APEXW_F32>(), s);
  const int64_t grid = ((int64_t)g.n * g.k + 255) / 256;
  hipLaunchKernelGGL(head_join_weight_kernel<DT>, dim3((unsigned)(grid < 4096 ? grid : 4096)), dim3(256), 0, s, g, state, partial);
}

void set_state(const HeadPlan& p, PackArgs& a, char* ws) {
  a.state = (HeadState*)ws, a.rows = (HeadRow*)(ws + p.at_rows), a.shift = (float*)(ws + p.at_shift);
}
// The weights, copied to whole chunks where they are not; rows packed
template <int DT> const uint16_t* launch_pack(const HeadPlan& p, PackArgs& a, const void* w, int64_t stride, char* ws, hipStream_t s) {
  set_state(p, a, ws);
  a.packed = (uint16_t*)(ws + p.at_x), a.w = (const uint16_t*)w, a.w_stride = stride;
  a.n = p.n, a.width = (int32_t)p.width, a.wide = (int32_t)p.wide, a.vocab = (int32_t)p.vocab;
  // about 1024 workgroups, of at least 4 rows
  const int64_t per = (p.n + 1023) / 1024;
  a.per = (int32_t)(per < 4 ? 4 : per);
  const int groups = p.n ? (int)((p.n + a.per - 1) / a.per) : 1;
  const uint16_t* from = (const uint16_t*)w;
  Pad weights{};
  int64_t copies = 0;
  if (p.copy_w) {
    uint16_t* at = (uint16_t*)(ws + p.at_w);
    int64_t step = 0;
    weights = pad(from, stride, step, p.vocab, p.vocab, (int32_t)p.width, at);
    copies = p.vocab * p.width / 2048 + 1;
  }
  hipLaunchKernelGGL(head_pack_kernel<DT>, dim3((unsigned)(groups + (copies < 8192 ? copies : 8192))), dim3(256), 0, s, a, weights,
                     groups);
  return from;
}

template <class F> void by_half(int32_t dtype, F&& f) {
  if (dtype == APEXW_BF16) f(std::integral_constant<int, APEXW_BF16>());
  else f(std::integral_constant<int, APEXW_F16>());
}

}  // namespace

extern "C" int64_t apexw_linear_cross_entropy_workspace(const void* weight, int64_t w_stride, int64_t n, int64_t width,
                                                        int64_t vocab, int32_t backward) {
  if (!head_ok(n, width, vocab)) return -APEXW_ERR_ARG;
  const HeadPlan p(weight, w_stride, n, width, vocab, backward != 0, backward & 1, backward & 2);
  return head_fits(p) ? p.bytes : -APEXW_ERR_SIZE;
}

extern "C" int apexw_linear_cross_entropy_forward(const void* x, int64_t x_stride, int64_t n, int64_t width,
                                                  const void* weight, int64_t w_stride, int64_t vocab, int32_t dtype,
                                                  const void* target, int32_t id_bytes, int64_t ignore_index, float* loss,
                                                  float* lse, int32_t reduction, float* total, void* workspace,
                                                  void* stream) {
  if (!head_ok(n, width, vocab) || x_stride < 0 || w_stride < 0 || (id_bytes != 4 && id_bytes != 8)) return APEXW_ERR_ARG;
  if (!weight || !workspace || (n > 0 && (!x || !target || !loss || !lse))) return APEXW_ERR_ARG;
  if (reduction < 0 || reduction > 2 || (reduction > 0 && !total)) return APEXW_ERR_ARG;
  if (dtype != APEXW_BF16 && dtype != APEXW_F16) return APEXW_ERR_DTYPE;
  if ((((uintptr_t)x | (uintptr_t)weight) & 1u) || ((uintptr_t)target & (id_bytes - 1)) || ((uintptr_t)workspace & 15u) ||
      (((uintptr_t)loss | (uintptr_t)lse | (uintptr_t)total) & 3u))
    return APEXW_ERR_ALIGN;
  const HeadPlan p(weight, w_stride, n, width, vocab, false, false, false);
  if (!head_fits(p)) return APEXW_ERR_SIZE;
  hipStream_t s = (hipStream_t)stream;
  char* ws = (char*)workspace;
  PackArgs pack{};
  pack.x = (const uint16_t*)x, pack.x_stride = x_stride, pack.target = target, pack.id64 = id_bytes == 8;
  pack.ignore = ignore_index, pack.loss = loss, pack.lse_out = lse;
  by_half(dtype, [&](auto d) {
    constexpr int DT = decltype(d)::value;
    ExpertArgs g = p.args(vocab);
    const FewTargets targets{(const uint32_t*)target, ignore_index, pack.id64, (int32_t)vocab};
    const bool few = n > 0 && n <= Small::BM && p.cut.shape == 0 && !p.copy_w && k_rows_ok(x, x_stride, width);
    const uint16_t* w = (const uint16_t*)weight;
    if (few) set_state(p, pack, ws);
    else w = launch_pack<DT>(p, pack, weight, w_stride, ws, s);
    if (n == 0) return;
    const HeadArgs h{pack.state, pack.rows, pack.shift, (float*)(ws + p.at_parts), p.parts_ld};
    if (few) {
      g.a = (const uint16_t*)x, g.lda = x_stride, g.b = w;
      hipLaunchKernelGGL(head_few_kernel<DT>, dim3(stream_grid<Small>((vocab + Small::BN - 1) / Small::BN)), dim3(Small::kThreads), 0, s,
                         g, FewSums{h, targets, pack.shift}, pack.state);
    } else {
      g.a = pack.packed, g.b = w, g.ends = &pack.state->count;
      launch_logits<DT>(g, p.cut.shape, Sums{h}, s);
    }
    const int64_t joins = (n + 15) / 16;
    const dim3 grid((unsigned)(joins < kJoins ? joins : kJoins), (unsigned)((joins + kJoins - 1) / kJoins));
    hipLaunchKernelGGL(head_join_kernel, grid, dim3(1024), 0, s, h, (int)p.parts(), few ? (int)n : 0, targets, loss, lse);
  });
  if (reduction) hipLaunchKernelGGL(head_total_kernel, dim3(1), dim3(1024), 0, s, pack.state, loss, n, (int)(reduction == 2), total);
  return hipGetLastError() == hipSuccess ? APEXW_OK : APEXW_ERR_LAUNCH;
}

extern "C" int apexw_linear_cross_entropy_backward(const float* dloss, int64_t dloss_stride, int32_t mean, const void* x,
                                                   int64_t x_stride, int64_t n, int64_t width, const void* weight,
                                                   int64_t w_stride, int64_t vocab, int32_t dtype, const void* target,
                                                   int32_t id_bytes, int64_t ignore_index, const float* lse, void* dx,
                                                   void* dw, void* workspace, void* stream) {
  if (!head_ok(n, width, vocab) || x_stride < 0 || w_stride < 0 || dloss_stride < 0 || (id_bytes != 4 && id_bytes != 8))
    return APEXW_ERR_ARG;
  if (!weight || !workspace || (n > 0 && (!x || !target || !dloss || !lse))) return APEXW_ERR_ARG;
  if (dtype != APEXW_BF16 && dtype != APEXW_F16) return APEXW_ERR_DTYPE;
  if ((((uintptr_t)x | (uintptr_t)weight | (uintptr_t)dx | (uintptr_t)dw) & 1u) || ((uintptr_t)target & (id_bytes - 1)) ||
      ((uintptr_t)workspace & 15u) || (((uintptr_t)dloss | (uintptr_t)lse) & 3u))
    return APEXW_ERR_ALIGN;
  if (!dx && !dw) return APEXW_OK;
  const HeadPlan p(weight, w_stride, n, width, vocab, true, dx != nullptr, dw != nullptr);
  if (!head_fits(p)) return APEXW_ERR_SIZE;
  hipStream_t s = (hipStream_t)stream;
  char* ws = (char*)workspace;
  PackArgs pack{};
  pack.x = (const uint16_t*)x, pack.x_stride = x_stride, pack.target = target, pack.id64 = id_bytes == 8;
  pack.ignore = ignore_index, pack.lse = lse, pack.dloss = dloss, pack.dloss_stride = dloss_stride, pack.dx = dx;
  pack.mean = mean != 0;
  by_half(dtype, [&](auto d) {
    constexpr int DT = decltype(d)::value;
    const uint16_t* w = launch_pack<DT>(p, pack, weight, w_stride, ws, s);
    const HeadArgs h{pack.state, pack.rows, pack.shift, nullptr, 0};
    uint16_t* G = (uint16_t*)(ws + p.at_g);
    float* sums = (float*)(ws + p.at_sums);
    for (int64_t v = 0; v < vocab; v += p.piece.cols) {
      const Piece& q = p.at_column(v);
      const uint16_t* wp = w + v * p.w_stride;
      if (n > 0) {
        ExpertArgs g = p.logits(q);
        g.a = pack.packed, g.b = wp, g.ends = &pack.state->count, g.out = G;
        launch_logits<DT>(g, q.logits.shape, Prob<DT>{h, (int32_t)v}, s);
        if (targets_apart(q.logits.shape))
          hipLaunchKernelGGL(head_targets_kernel<DT>, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, h, (int)v, (int)q.cols, G,
                             p.piece_ld);
      }
      if (dw) {
        ExpertArgs g = p.dw(q);
        g.a = G, g.b = pack.packed, g.ends = &pack.state->count, g.out = (uint16_t*)dw + v * width;
        launch_dw<DT>(g, q.dw.shape, pack.state, (float*)(ws + p.at_dw), s);
      }
      if (dx && n > 0) {
        ExpertArgs g = p.dx(q);
        g.a = G, g.b = wp, g.ends = &pack.state->count, g.out = sums;
        launch_dx<DT>(g, q.dx.shape, v > 0, s);
      }
    }
    if (dx && n > 0) {
      const int64_t grid = (n * ((width + 3) / 4) + 255) / 256;
      hipLaunchKernelGGL(head_dx_kernel<DT>, dim3((unsigned)(grid < 8192 ? grid : 8192)), dim3(256), 0, s, h,
                         sums, n * width, p.dx(p.piece).splits, (int)width, (uint16_t*)dx);
    }
  });
  return hipGetLastError() == hipSuccess ? APEXW_OK : APEXW_ERR_LAUNCH;
}
