// Tokens sorted by expert and back, and the embedding, with their gradients (gfx950).
//
// Choice c = t k + j of token t names expert e_c; those in [0, experts) get rows in the order of (e_c, c):
//   place[c]: the choice's row, -1 for one that no expert takes;  source[r]: the row's choice, -1 behind the last end
//   dispatch      rows_r = x_{source_r / k}                 its gradient   dx_t = sum_j drows_place(t, j)
//   combine       o_t = sum_j w_tj y_place(t, j)            its gradient   dy_r = w_source do_{source / k},  dw_tj = <do_t, y_place(t, j)>
//   embedding     y_t = s W_id(t)                           its gradient   dW_v = s sum over id(t) = v of dy_t
// Sums are fp32, rounded once, in an order that the sizes and ids alone set.
//
// All of it is bound by memory.  Dispatch, combine and its gradient go token by token: a token's row is read (written)
// once and its k rows by expert, whole, wherever they lie.
//
// Measured, kernels alone (a large copy: 4.7 TB/s):
//   order and dispatch, 16384 tokens x 2 of 8 experts, 4096 bf16     4.7 + 5.1 and 66 us   6.1 TB/s
//   the same, 16 x 2 of 64, 2048 bf16                                3.7 and 3.6 us
//   combine, 8192 tokens x 8, 2048 bf16                              59 us   5.1 TB/s
//   combine's gradient, 4097 tokens x 3, 1021 fp32                   26 us   4.4 TB/s
//   embedding, 16384 of 128256 x 4096 bf16                           34 us   (ids that recur are read from the cache)
//   its gradient, 16384 tokens, 50257 x 768 bf16                     sort 19, blocks 6.6, rows 21 us
//   the same, 65536 tokens, 128256 x 4096 bf16                       sort 27, blocks 71, rows 285 us   4.1 TB/s in all
// (The blocks' launch of the last one moves 130 MB, but the memory is still writing the last call's 1 GB.)
#include <type_traits>

#include "chunks.h"
#include "sort.h"

int apexw_cu_count();

namespace {

// ---------------------------------------------------------------------------
// Order
// ---------------------------------------------------------------------------

template <int kItems> __global__ __launch_bounds__(kSortThreads) void order_small_kernel(SortArgs a) { sort_small<true, kItems>(a); }

// ends[e] = items of keys up to e, for orders that took more than one pass
__global__ __launch_bounds__(256) void order_ends_kernel(const u32x2* __restrict__ sorted, int n, uint32_t experts, int32_t* ends) {
  for (uint32_t e = blockIdx.x * 256u + threadIdx.x; e < experts; e += gridDim.x * 256u) {
    int lo = 0, hi = n;
    while (lo < hi) {
      const int mid = lo + (hi - lo) / 2;
      if (sorted[mid][0] <= e) lo = mid + 1;
      else hi = mid;
    }
    ends[e] = lo;
  }
}

// ---------------------------------------------------------------------------
// Dispatch and combine
// ---------------------------------------------------------------------------

// A grid's first dimension times 256 threads has to stay below 2^32, so many workgroups go along two
constexpr int64_t kAcross = 1 << 20;
APEXW_DEV int64_t group_of() { return (int64_t)blockIdx.y * gridDim.x + blockIdx.x; }
dim3 groups_grid(int64_t groups) {
  return dim3((unsigned)(groups < kAcross ? groups : kAcross), (unsigned)((groups + kAcross - 1) / kAcross));
}

// T threads (a power of two, up to 256) share a token
struct TokenArgs {
  const void *x, *y;           // rows by token, rows by expert
  int64_t x_stride, y_stride;
  const int32_t *source, *place;
  const void* weight;
  void *out, *dweight;
  int64_t tokens;
  int32_t k, width, log_t;
};
constexpr int kWG = 256;

struct Token {
  int64_t t;
  int lane, step;
  bool here;
  __device__ __forceinline__ explicit Token(const TokenArgs& a)
      : t(group_of() * (kWG >> a.log_t) + (threadIdx.x >> a.log_t)), lane(threadIdx.x & ((1 << a.log_t) - 1)),
        step(1 << a.log_t), here(t < a.tokens) {}
};
APEXW_DEV int64_t row_of(const TokenArgs& a, int64_t choice) {   // -1 for any place that is no row
  const int32_t p = APEXW_GLOBAL(const int32_t, a.place)[choice];
  return p >= 0 && p < a.tokens * a.k ? p : -1;
}

// Zeros in the rows behind the last end among rows t k .. t k + k - 1
template <int DT> APEXW_DEV void zero_spare(const TokenArgs& a, const Token& me, const RowChunks<DT>& row, void* rows) {
  for (int j = 0; j < a.k; ++j) {
    const int64_t r = me.t * a.k + j;
    if (APEXW_GLOBAL(const int32_t, a.source)[r] >= 0) continue;
    for (int c = me.lane; c < row.count; c += me.step) row.store(row_at<DT>(rows, r * a.width), c, u32x4{0u, 0u, 0u, 0u});
  }
}

template <int DT> __global__ __launch_bounds__(kWG) void dispatch_kernel(TokenArgs a) {
  const Token me(a);
  if (!me.here) return;
  const RowChunks<DT> row(a.width);
  const void* x = row_at<DT>(a.x, me.t * a.x_stride);
  constexpr int U = 4;
  for (int c0 = me.lane; c0 < row.count; c0 += U * me.step) {
    u32x4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (c0 + u * me.step < row.count) v[u] = row.load(x, c0 + u * me.step);
    for (int j = 0; j < a.k; ++j) {
      const int64_t p = row_of(a, me.t * a.k + j);
      if (p < 0) continue;
      void* to = row_at<DT>(a.out, p * a.width);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (c0 + u * me.step < row.count) row.store(to, c0 + u * me.step, v[u]);
    }
  }
  zero_spare<DT>(a, me, row, a.out);
}

// WD: the weights' type, or -1 without
template <int DT, int WD> __global__ __launch_bounds__(kWG) void combine_kernel(TokenArgs a) {
  const Token me(a);
  if (!me.here) return;
  const RowChunks<DT> row(a.width);
  constexpr int KU = 8, V = kVec<DT>;
  for (int c = me.lane; c < row.count; c += me.step) {
    float sum[V] = {};
    for (int j0 = 0; j0 < a.k; j0 += KU) {
      u32x4 v[KU];
      float w[KU];
      bool has[KU];
#pragma unroll
      for (int j = 0; j < KU; ++j) {
        const int64_t choice = me.t * a.k + j0 + j, p = j0 + j < a.k ? row_of(a, choice) : -1;
        has[j] = p >= 0;
        if (!has[j]) continue;
        v[j] = row.load(row_at<DT>(a.y, p * a.y_stride), c);
        if constexpr (WD >= 0) w[j] = load1<WD>(a.weight, choice);
      }
#pragma unroll
      for (int j = 0; j < KU; ++j) {
        if (!has[j]) continue;
        float x[V];
        values<DT>(v[j], x);
#pragma unroll
        for (int i = 0; i < V; ++i) sum[i] = WD >= 0 ? fmaf(w[j], x[i], sum[i]) : sum[i] + x[i];
      }
    }
    row.store(row_at<DT>(a.out, me.t * a.width), c, rounded<DT>(sum));
  }
}

// x: the gradient of the combined rows.  Two choices at a time: 4 take 102 registers, half of the waves (4097 x 1021 fp32, 3
// choices, 34 us, by two 26)
template <int DT, int WD> __global__ __launch_bounds__(kWG) void combine_backward_kernel(TokenArgs a) {
  const Token me(a);
  const RowChunks<DT> row(a.width);
  constexpr int KU = 2, V = kVec<DT>;
  __shared__ float parts[kWG / 64][KU];
  const void* x = row_at<DT>(a.x, me.here ? me.t * a.x_stride : 0);
  for (int j0 = 0; j0 < a.k; j0 += KU) {
    int64_t p[KU];
    float w[KU], dot[KU] = {};
#pragma unroll
    for (int j = 0; j < KU; ++j) {
      const int64_t choice = me.t * a.k + j0 + j;
      p[j] = me.here && j0 + j < a.k ? row_of(a, choice) : -1;
      w[j] = p[j] >= 0 ? load1<WD>(a.weight, choice) : 0.0f;
    }
    if (me.here)
      for (int c = me.lane; c < row.count; c += me.step) {
        const u32x4 d = row.load(x, c);
        u32x4 v[KU];
        if (a.dweight) {
#pragma unroll
          for (int j = 0; j < KU; ++j)
            if (p[j] >= 0) v[j] = row.load(row_at<DT>(a.y, p[j] * a.y_stride), c);
        }
        float dx[V];
        values<DT>(d, dx);
        if (a.out) {
#pragma unroll
          for (int j = 0; j < KU; ++j) {
            if (p[j] < 0) continue;
            float g[V];
#pragma unroll
            for (int i = 0; i < V; ++i) g[i] = w[j] * dx[i];
            row.store(row_at<DT>(a.out, p[j] * a.width), c, rounded<DT>(g));
          }
        }
        if (a.dweight) {
          const int skip = row.skip(c);
#pragma unroll
          for (int j = 0; j < KU; ++j) {
            if (p[j] < 0) continue;
            float y[V];
            values<DT>(v[j], y);
#pragma unroll
            for (int i = 0; i < V; ++i) dot[j] = i >= skip && i < a.width ? fmaf(dx[i], y[i], dot[j]) : dot[j];
          }
        }
      }
    if (!a.dweight) continue;
#pragma unroll
    for (int j = 0; j < KU; ++j)
      for (int off = me.step < 64 ? me.step / 2 : 32; off > 0; off >>= 1) dot[j] += __shfl_xor(dot[j], off, 64);
    if (me.step > 64) {   // the four waves of one token
      if (lane_id() == 0)
#pragma unroll
        for (int j = 0; j < KU; ++j) parts[threadIdx.x >> 6][j] = dot[j];
      __syncthreads();
#pragma unroll
      for (int j = 0; j < KU; ++j) dot[j] = (parts[0][j] + parts[1][j]) + (parts[2][j] + parts[3][j]);
      __syncthreads();
    }
    if (me.here && me.lane == 0)
#pragma unroll
      for (int j = 0; j < KU; ++j)
        if (j0 + j < a.k) store1<WD>(a.dweight, me.t * a.k + j0 + j, rnd<WD>(p[j] >= 0 ? dot[j] : 0.0f));
  }
  if (me.here && a.out) zero_spare<DT>(a, me, row, a.out);
}

// ---------------------------------------------------------------------------
// Embedding
// ---------------------------------------------------------------------------

struct EmbeddingArgs {
  const void *ids, *w;      // w: the table, or dy
  void* out;
  int64_t n, stride;        // rows; of w
  uint32_t vocab;
  int32_t wide, width, log_t;
  float scale;
  const u32x2* sorted;      // (id, token)
  int32_t* many;            // the number of ids of many tokens, and, behind 4 of them, which they are
  int32_t* ranges;          // [vocab][2]: where an id's tokens begin and end among the sorted, 0 0 for none
  float* blocks;            // sums of whole blocks of 2^log_block sorted tokens of one id
  int32_t log_block;
};

template <int DT> APEXW_DEV u32x4 scaled(u32x4 w, float scale) {
  float x[kVec<DT>];
  values<DT>(w, x);
#pragma unroll
  for (int i = 0; i < kVec<DT>; ++i) x[i] *= scale;
  return rounded<DT>(x);
}

template <int DT> __global__ __launch_bounds__(kWG) void embedding_kernel(EmbeddingArgs a) {
  const int64_t t = group_of() * (kWG >> a.log_t) + (threadIdx.x >> a.log_t);
  if (t >= a.n) return;
  const RowChunks<DT> row(a.width);
  const int step = 1 << a.log_t, lane = threadIdx.x & (step - 1);
  const int64_t id = a.wide ? APEXW_GLOBAL(const int64_t, a.ids)[t] : APEXW_GLOBAL(const int32_t, a.ids)[t];
  const bool has = (uint64_t)id < a.vocab;
  const void* from = row_at<DT>(a.w, has ? id * a.stride : 0);
  void* to = row_at<DT>(a.out, t * a.width);
  constexpr int U = 4;
  for (int c0 = lane; c0 < row.count; c0 += U * step) {
    u32x4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      v[u] = u32x4{0u, 0u, 0u, 0u};
      if (has && c0 + u * step < row.count) v[u] = row.load(from, c0 + u * step);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (c0 + u * step < row.count) row.store(to, c0 + u * step, scaled<DT>(v[u], a.scale));
  }
}

template <int kItems> __global__ __launch_bounds__(kSortThreads) void embedding_sort_kernel(SortArgs a) {
  if (blockIdx.x) return sort_clear(a, blockIdx.x - 1, gridDim.x - 1);
  sort_small<false, kItems>(a);
}

// sum += the rows of sorted tokens [from, to), U in flight, chunk c of each
template <int DT, int U> APEXW_DEV void add_rows(const EmbeddingArgs& a, const RowChunks<DT>& row, int c, int from, int to,
                                          float (&sum)[kVec<DT>]) {
  if (c >= row.count) return;
  for (int p = from; p < to; p += U) {
    uint32_t token[U];
    u32x4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (p + u < to) token[u] = a.sorted[p + u][1];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (p + u < to) v[u] = row.load(row_at<DT>(a.w, token[u] * a.stride), c);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (p + u < to) {
        float x[kVec<DT>];
        values<DT>(v[u], x);
#pragma unroll
        for (int i = 0; i < kVec<DT>; ++i) sum[i] += x[i];
      }
  }
}

// The four waves' sums of a chunk, added up by the first one; all threads call it
template <int V> APEXW_DEV void join_waves(float (&sum)[V], float (*lds)[64][V]) {
  const int wave = threadIdx.x >> 6, lane = lane_id();
#pragma unroll
  for (int i = 0; i < V; ++i) lds[wave][lane][i] = sum[i];
  __syncthreads();
  if (wave == 0) {
#pragma unroll
    for (int i = 0; i < V; ++i) sum[i] = (lds[0][lane][i] + lds[1][lane][i]) + (lds[2][lane][i] + lds[3][lane][i]);
  }
  __syncthreads();
}

// part q of four of [from, to)
struct Part {
  int from, to;
  __device__ __forceinline__ Part(int f, int t, int q) {
    const int len = (t - f + 3) / 4;
    from = f + q * len, to = from + len;
    from = from < t ? from : t, to = to < t ? to : t;
  }
};

// Ids of more tokens than this are summed by the four waves of a workgroup
constexpr int kMany = 48, kManyGroups = 512;

// Where each id's tokens lie, which ids have many, and the sums of the whole blocks of one id: 64 chunks of columns a
// workgroup
template <int DT> __global__ __launch_bounds__(kWG) void embedding_blocks_kernel(EmbeddingArgs a) {
  constexpr int V = kVec<DT>;
  __shared__ float lds[4][64][V];
  const int n = (int)a.n, first = blockIdx.x << a.log_block, size = 1 << a.log_block;
  if (blockIdx.y == 0)
    for (int i = first + threadIdx.x; i < n && i < first + size; i += kWG) {
      const uint32_t key = a.sorted[i][0];
      if (key >= a.vocab) continue;
      if (i == 0 || a.sorted[i - 1][0] != key) {
        a.ranges[2 * (int64_t)key] = i;
        // (the list's order is of no consequence)
        if (i + kMany < n && a.sorted[i + kMany][0] == key) a.many[4 + atomicAdd(a.many, 1)] = (int32_t)key;
      }
      if (i == n - 1 || a.sorted[i + 1][0] != key) a.ranges[2 * (int64_t)key + 1] = i + 1;
    }
  if (n - first < size) return;
  const uint32_t key = a.sorted[first][0];
  if (key >= a.vocab || a.sorted[first + size - 1][0] != key) return;
  const RowChunks<DT> row(a.width);
  const int c = blockIdx.y * 64 + lane_id();
  float sum[V] = {};
  const Part p(first, first + size, threadIdx.x >> 6);
  add_rows<DT, 8>(a, row, c, p.from, p.to, sum);
  join_waves<V>(sum, lds);
  if (threadIdx.x < 64 && c < row.count) {
    float* to = a.blocks + (int64_t)blockIdx.x * row.count * V + c * V;
#pragma unroll
    for (int i = 0; i < V; ++i) to[i] = sum[i];
  }
}

// part `q` of `of` of the sum over sorted tokens [lo, hi): whole blocks, where some lie in it, and what is around them
template <int DT> APEXW_DEV void add_range(const EmbeddingArgs& a, const RowChunks<DT>& row, int c, int lo, int hi, int q,
                                           int of, float (&sum)[kVec<DT>]) {
  constexpr int V = kVec<DT>;
  const int size = 1 << a.log_block, b0 = (lo + size - 1) >> a.log_block, b1 = hi >> a.log_block;
  const auto rows = [&](int from, int to) {
    if (of == 1) return add_rows<DT, 4>(a, row, c, from, to, sum);
    const Part p(from, to, q);
    add_rows<DT, 4>(a, row, c, p.from, p.to, sum);
  };
  if (b0 >= b1) return rows(lo, hi);
  rows(lo, b0 << a.log_block);
  int from = b0, to = b1;
  if (of > 1) {
    const Part p(b0, b1, q);
    from = p.from, to = p.to;
  }
  if (c < row.count) {
    const float* p = a.blocks + (int64_t)from * row.count * V + c * V;
#pragma unroll 4
    for (int b = from; b < to; ++b, p += (int64_t)row.count * V)
#pragma unroll
      for (int i = 0; i < V; ++i) sum[i] += p[i];
  }
  rows(b1 << a.log_block, hi);
}

// A row of the gradient, chunk c
template <int DT, int OD> APEXW_DEV void write_sum(const EmbeddingArgs& a, const RowChunks<DT>& row, int64_t v, int c, float (&sum)[kVec<DT>]) {
  constexpr int V = kVec<DT>;
  if (c >= row.count) return;
#pragma unroll
  for (int i = 0; i < V; ++i) sum[i] *= a.scale;
  if constexpr (OD == DT) {
    row.store(row_at<OD>(a.out, v * a.width), c, rounded<DT>(sum));
  } else {
    const int at = row.begin(c);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const u32x4 w = {__float_as_uint(sum[4 * q]), __float_as_uint(sum[4 * q + 1]), __float_as_uint(sum[4 * q + 2]),
                       __float_as_uint(sum[4 * q + 3])};
      if (a.width >= V) chunk_to<OD>(a.out, v * a.width + at + 4 * q, w);
      else part_to<OD>(a.out, v * a.width + 4 * q, a.width - 4 * q, w);
    }
  }
}

// Few tokens, whose sort clears the gradient beside it: a workgroup has 64 chunks of columns of the id that a token is
// the first one of, a part of its tokens a wave.  (50257 x 768 bf16, 1 to 1024 tokens 15 to 18 us, by the other kernels
// 25 to 32; 2048 tokens 25 and 33, but 87 and 35 where all are of one id.)
constexpr int kFewTokens = 1024;
template <int DT, int OD> __global__ __launch_bounds__(kWG) void embedding_few_kernel(EmbeddingArgs a) {
  constexpr int V = kVec<DT>;
  __shared__ float lds[4][64][V];
  const int lo = blockIdx.x, n = (int)a.n;
  const uint32_t key = a.sorted[lo][0];
  if (key >= a.vocab || (lo > 0 && a.sorted[lo - 1][0] == key)) return;
  int hi = lo;
  for (int i = lo; i < n; i += kWG) {
    const int more = __syncthreads_count(i + (int)threadIdx.x < n && a.sorted[i + threadIdx.x][0] == key);
    hi += more;
    if (more < kWG) break;
  }
  const RowChunks<DT> row(a.width);
  const int c = blockIdx.y * 64 + lane_id();
  float sum[V] = {};
  const Part p(lo, hi, threadIdx.x >> 6);
  add_rows<DT, 16>(a, row, c, p.from, p.to, sum);
  join_waves<V>(sum, lds);
  if (threadIdx.x < 64) write_sum<DT, OD>(a, row, key, c, sum);
}

// The gradient's rows: up to 64 of them a workgroup, every (number of workgroups)th, so that frequent words, which have
// neighbouring ids, go to different ones.  A row is taken 64 chunks of columns a wave, narrow rows several a wave.  The
// first kManyGroups workgroups take the ids of many tokens, 64 chunks each, a part of the tokens a wave: one that met
// such an id among its rows would end long after the others (65536 tokens, a tenth of them one id, 128256 x 4096: 511 us).
template <int DT, int OD> __global__ __launch_bounds__(kWG) void embedding_grad_kernel(EmbeddingArgs a, int rows) {
  constexpr int V = kVec<DT>;
  const RowChunks<DT> row(a.width);
  const int slabs = (row.count + 63) / 64, wave = uniform(threadIdx.x >> 6), lane = lane_id();
  const auto write = [&](int64_t v, int c, float (&sum)[V]) { write_sum<DT, OD>(a, row, v, c, sum); };
  if (blockIdx.x < kManyGroups) {
    __shared__ float lds[4][64][V];
    const int64_t units = (int64_t)a.many[0] * slabs;
    for (int64_t u = blockIdx.x; u < units; u += kManyGroups) {
      const int64_t v = a.many[4 + u / slabs];
      const int c = (int)(u % slabs) * 64 + lane;
      float sum[V] = {};
      add_range<DT>(a, row, c, a.ranges[2 * v], a.ranges[2 * v + 1], wave, 4, sum);
      join_waves<V>(sum, lds);
      if (wave == 0) write(v, c, sum);
    }
    return;
  }
  __shared__ int range[64][3];   // of a row: its tokens among the sorted, and the first one
  const int64_t groups = gridDim.x - kManyGroups, group = blockIdx.x - kManyGroups;
  if ((int)threadIdx.x < rows) {
    const int64_t v = group + threadIdx.x * groups;
    int lo = 0, hi = 0;
    if (v < a.vocab) lo = a.ranges[2 * v], hi = a.ranges[2 * v + 1];
    range[threadIdx.x][0] = lo, range[threadIdx.x][1] = hi;
    range[threadIdx.x][2] = hi > lo ? (int)a.sorted[lo][1] : 0;
  }
  __syncthreads();
  const auto light = [&](int64_t v, int lo, int hi, int token, int c) {
    float sum[V] = {};
    if (hi - lo == 1) {
      if (c < row.count) values<DT>(row.load(row_at<DT>(a.w, token * a.stride), c), sum);
    } else if (hi > lo) {
      add_range<DT>(a, row, c, lo, hi, 0, 1, sum);
    }
    write(v, c, sum);
  };
  if (slabs == 1) {   // 2^log_t threads a row
    const int per = 64 >> a.log_t, c = lane & ((1 << a.log_t) - 1);
    for (int r = wave * per + (lane >> a.log_t); r < rows; r += 4 * per) {
      const int64_t v = group + r * groups;
      if (v >= a.vocab) break;
      if (range[r][1] - range[r][0] <= kMany) light(v, range[r][0], range[r][1], range[r][2], c);
    }
    return;
  }
  if (slabs < 4) {
    for (int u = wave; u < rows * slabs; u += 4) {
      const int r = u / slabs, c = (u - r * slabs) * 64 + lane;
      const int64_t v = group + r * groups;
      if (v >= a.vocab) break;
      const int lo = range[r][0], hi = range[r][1];
      if (hi - lo > kMany) continue;
      float sum[V] = {};
      if (hi > lo) add_range<DT>(a, row, c, lo, hi, 0, 1, sum);
      write(v, c, sum);
    }
    return;
  }
  for (int r = 0; r < rows; ++r) {
    const int64_t v = group + r * groups;
    if (v >= a.vocab) break;
    const int lo = range[r][0], hi = range[r][1], token = uniform(range[r][2]);   // (scalar loads of the sorted are slower)
    if (hi - lo > kMany) continue;
    int s = wave;
    for (; hi - lo <= 1 && s + 4 < slabs; s += 8) {   // two at once
      const int c0 = s * 64 + lane, c1 = c0 + 256;
      float x[V] = {}, y[V] = {};
      if (hi > lo) {
        const void* from = row_at<DT>(a.w, token * a.stride);
        const u32x4 p = row.load(from, c0), q = row.load(from, c1 < row.count ? c1 : c0);
        values<DT>(p, x), values<DT>(q, y);
      }
      write(v, c0, x);
      write(v, c1, y);
    }
    for (; s < slabs; s += 4) light(v, lo, hi, token, s * 64 + lane);
  }
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------

// (a row of the embedding's gradient is up to 65535 slabs of 64 chunks)
bool rows_ok(int64_t n, int64_t width) { return n >= 0 && n <= INT32_MAX - 65536 && width > 0 && width <= APEXW_ROW_WIDTH; }
int64_t aligned(int64_t bytes) { return (bytes + 255) / 256 * 256; }

// The workspace of a sort: counts, and the pairs of passes that follow another or are wanted sorted
struct SortSpace {
  int64_t counts, pairs, bytes;
  SortSpace(const SortArgs& a, bool wanted) {
    const bool small = a.n <= kSmall;
    counts = small ? 0 : aligned(((int64_t)(sort_groups(a.n) + 1) << a.bits) * 4);
    pairs = aligned((int64_t)a.n * 8);
    const int lists = (wanted ? 1 : 0) + (small ? 0 : a.passes - 1 < 2 ? a.passes - 1 : 2);
    bytes = counts + pairs * (lists > 2 ? 2 : lists);
  }
};

SortArgs sort_args(const void* ids, int32_t id_bytes, int64_t n, uint32_t limit) {
  SortArgs a{};
  a.ids = ids, a.wide = id_bytes == 8, a.n = (int32_t)n, a.limit = limit;
  sort_digits(a);
  return a;
}

// More than kSmall items: the passes, from one list to the other; the sorted pairs where they are wanted
template <bool kOrder, int kItems> const u32x2* launch_passes(SortArgs a, const SortSpace& space, bool wanted, char* ws, hipStream_t s) {
  a.counts = (uint32_t*)ws;
  u32x2* lists[2] = {(u32x2*)(ws + space.counts), (u32x2*)(ws + space.counts + space.pairs)};
  const dim3 grid((unsigned)sort_groups(a.n)), block(kSortThreads);
  for (int pass = 0; pass < a.passes; ++pass) {
    const bool last = pass == a.passes - 1;
    a.from = pass ? lists[(pass - 1) & 1] : nullptr;
    a.to = last && !wanted ? nullptr : lists[pass & 1];
    if (pass == 0) hipLaunchKernelGGL((sort_count_kernel<true, kItems>), grid, block, 0, s, a, pass);
    else hipLaunchKernelGGL((sort_count_kernel<false, kItems>), grid, block, 0, s, a, pass);
    if (grid.x > kScan)
      hipLaunchKernelGGL(sort_scan_kernel, dim3((unsigned)((1 << a.bits) + 63) / 64), dim3(1024), 0, s, a.counts, (int)grid.x, 1 << a.bits);
    if (kOrder && last) {
      if (pass == 0) hipLaunchKernelGGL((sort_place_kernel<true, kOrder, kItems>), grid, block, 0, s, a, pass);
      else hipLaunchKernelGGL((sort_place_kernel<false, kOrder, kItems>), grid, block, 0, s, a, pass);
    } else {
      if (pass == 0) hipLaunchKernelGGL((sort_place_kernel<true, false, kItems>), grid, block, 0, s, a, pass);
      else hipLaunchKernelGGL((sort_place_kernel<false, false, kItems>), grid, block, 0, s, a, pass);
    }
  }
  return a.to;
}
template <bool kOrder> const u32x2* launch_sort(const SortArgs& a, const SortSpace& space, bool wanted, char* ws, hipStream_t s) {
  if (sort_items(a.n) == kFew) return launch_passes<kOrder, kFew>(a, space, wanted, ws, s);
  return launch_passes<kOrder, kMost>(a, space, wanted, ws, s);
}

// Threads of a row: a wave or less, or four where a row has a chunk for each of their threads.  (us with one and with
// four, k choices, bf16: combine's gradient of 16384 x 768, k = 1, 16.1 and 31.5, 8192 x 1536, k = 2, 22 and 25, 8192 x 2048,
// k = 8, 126 and 119; dispatch of 16384 x 768 10.2 and 15.6; combine of 8192 x 2048, k = 8, 76 and 59.)
int log_threads(int64_t width, int32_t dtype, bool four_waves) {
  const int64_t chunks = (width + (dtype == APEXW_F32 ? 3 : 7)) / (dtype == APEXW_F32 ? 4 : 8);
  int log_t = 4;
  while (log_t < 6 && (1 << log_t) < chunks) ++log_t;
  return four_waves && chunks >= kWG ? 8 : log_t;
}
TokenArgs token_args(int64_t tokens, int32_t k, int64_t width, int32_t dtype, const int32_t* source, const int32_t* place) {
  TokenArgs a{};
  a.tokens = tokens, a.k = k, a.width = (int32_t)width, a.source = source, a.place = place;
  a.log_t = log_threads(width, dtype, true);
  return a;
}
dim3 token_grid(const TokenArgs& a) {
  const int64_t per = kWG >> a.log_t;
  return groups_grid((a.tokens + per - 1) / per);
}
bool tokens_ok(int64_t tokens, int32_t k, int64_t width) {
  return tokens >= 0 && k > 0 && rows_ok(tokens, width) && tokens <= (INT32_MAX - 65536) / k;
}
int launched() { return hipGetLastError() == hipSuccess ? APEXW_OK : APEXW_ERR_LAUNCH; }

// f(rows' type, weights' type): the same, or fp32
template <class F> int by_types(int32_t dtype, int32_t w_dtype, F&& f) {
  if (w_dtype != dtype && w_dtype != APEXW_F32) return APEXW_ERR_DTYPE;
  const bool ok = by_row_type(dtype, [&](auto d) {
    if (w_dtype == APEXW_F32) f(d, std::integral_constant<int, APEXW_F32>());
    else f(d, d);
  });
  return ok ? APEXW_OK : APEXW_ERR_DTYPE;
}

// Rows of a gradient: 64 to a workgroup of 256 threads, fewer than 2^32 in all
constexpr int64_t kMostWords = 1 << 29;

// Workgroups that clear, at most (with 2048 in a loop 1 GB takes 226 us, with one for each 32 KB 187)
constexpr int64_t kClears = 1 << 20;

struct GradPlan {
  SortArgs sort;
  SortSpace space;
  int log_block;
  int64_t many, ranges, blocks, bytes;
  GradPlan(const void* ids, int32_t id_bytes, int64_t n, uint32_t vocab, int64_t width)
      : sort(sort_args(ids, id_bytes, n, vocab)), space(sort, true) {
    // a row's sum is over up to twice a block's tokens and one sum for each block
    log_block = n <= 32768 ? 6 : n <= 131072 ? 7 : 8;
    const bool few = n <= kFewTokens;
    many = few ? 0 : aligned(16 + n / kMany * 4);
    ranges = few ? 0 : aligned((int64_t)vocab * 8);
    blocks = few ? 0 : aligned((n >> log_block) * (width + 8) * 4);
    bytes = space.bytes + many + ranges + blocks;
  }
};

}  // namespace

extern "C" int64_t apexw_expert_order_workspace(int64_t choices, int32_t experts) {
  if (!rows_ok(choices, 1) || experts <= 0 || experts > INT32_MAX - 1) return -APEXW_ERR_ARG;
  const SortArgs a = sort_args(nullptr, 4, choices, (uint32_t)experts);
  return SortSpace(a, a.passes > 1).bytes;
}

extern "C" int apexw_expert_order(const void* expert, int32_t id_bytes, int64_t choices, int32_t experts, int32_t* source,
                                  int32_t* place, int32_t* ends, void* workspace, void* stream) {
  if (!ends || !rows_ok(choices, 1) || experts <= 0 || experts > INT32_MAX - 1 || (id_bytes != 4 && id_bytes != 8))
    return APEXW_ERR_ARG;
  if (choices > 0 && (!expert || !source || !place)) return APEXW_ERR_ARG;
  if (((uintptr_t)expert & (id_bytes - 1)) || (((uintptr_t)source | (uintptr_t)place | (uintptr_t)ends) & 3u) ||
      ((uintptr_t)workspace & 15u))
    return APEXW_ERR_ALIGN;
  SortArgs a = sort_args(expert, id_bytes, choices, (uint32_t)experts);
  const bool wanted = a.passes > 1;
  const SortSpace space(a, wanted);
  if (space.bytes > 0 && !workspace) return APEXW_ERR_ARG;
  hipStream_t s = (hipStream_t)stream;
  a.source = source, a.place = place, a.ends = ends;
  const u32x2* sorted = nullptr;
  if (a.n <= kSmall) {
    sorted = a.to = wanted ? (u32x2*)workspace : nullptr;
    if (a.n <= kFew * kSortThreads) hipLaunchKernelGGL(order_small_kernel<kFew>, dim3(1), dim3(kSortThreads), 0, s, a);
    else hipLaunchKernelGGL(order_small_kernel<kMost>, dim3(1), dim3(kSortThreads), 0, s, a);
  } else {
    sorted = launch_sort<true>(a, space, wanted, (char*)workspace, s);
  }
  if (wanted) {
    const int64_t grid = ((int64_t)experts + 255) / 256;
    hipLaunchKernelGGL(order_ends_kernel, dim3((unsigned)(grid < 1024 ? grid : 1024)), dim3(256), 0, s, sorted, a.n,
                       (uint32_t)experts, ends);
  }
  return launched();
}

extern "C" int apexw_expert_dispatch(const void* x, int64_t x_stride, int64_t tokens, int32_t k, int64_t width,
                                     int32_t dtype, const int32_t* source, const int32_t* place, void* rows,
                                     void* stream) {
  if (!tokens_ok(tokens, k, width) || x_stride < 0) return APEXW_ERR_ARG;
  if (tokens > 0 && (!x || !source || !place || !rows)) return APEXW_ERR_ARG;
  if (row_misaligned(x, dtype) || row_misaligned(rows, dtype) || (((uintptr_t)source | (uintptr_t)place) & 3u))
    return APEXW_ERR_ALIGN;
  TokenArgs a = token_args(tokens, k, width, dtype, source, place);
  a.x = x, a.x_stride = x_stride, a.out = rows;
  const bool ok = by_row_type(dtype, [&](auto d) {
    if (tokens > 0) hipLaunchKernelGGL(dispatch_kernel<decltype(d)::value>, token_grid(a), dim3(kWG), 0, (hipStream_t)stream, a);
  });
  return ok ? launched() : APEXW_ERR_DTYPE;
}

extern "C" int apexw_expert_combine(const void* y, int64_t y_stride, int64_t tokens, int32_t k, int64_t width,
                                    int32_t dtype, const int32_t* place, const void* weight, int32_t w_dtype, void* out,
                                    void* stream) {
  if (!tokens_ok(tokens, k, width) || y_stride < 0) return APEXW_ERR_ARG;
  if (tokens > 0 && (!y || !place || !out)) return APEXW_ERR_ARG;
  if (row_misaligned(y, dtype) || row_misaligned(out, dtype) || row_misaligned(weight, w_dtype) || ((uintptr_t)place & 3u))
    return APEXW_ERR_ALIGN;
  TokenArgs a = token_args(tokens, k, width, dtype, nullptr, place);
  a.y = y, a.y_stride = y_stride, a.weight = weight, a.out = out;
  const int st = by_types(dtype, weight ? w_dtype : dtype, [&](auto d, auto w) {
    constexpr int DT = decltype(d)::value, WD = decltype(w)::value;
    if (tokens == 0) return;
    if (weight) hipLaunchKernelGGL((combine_kernel<DT, WD>), token_grid(a), dim3(kWG), 0, (hipStream_t)stream, a);
    else hipLaunchKernelGGL((combine_kernel<DT, -1>), token_grid(a), dim3(kWG), 0, (hipStream_t)stream, a);
  });
  return st ? st : launched();
}

extern "C" int apexw_expert_combine_backward(const void* dout, int64_t dout_stride, const void* y, int64_t y_stride,
                                             int64_t tokens, int32_t k, int64_t width, int32_t dtype,
                                             const int32_t* source, const int32_t* place, const void* weight,
                                             int32_t w_dtype, void* dy, void* dweight, void* stream) {
  if (!tokens_ok(tokens, k, width) || dout_stride < 0 || y_stride < 0) return APEXW_ERR_ARG;
  if (tokens > 0 && (!dout || !source || !place || !weight || (dweight && !y))) return APEXW_ERR_ARG;
  if (row_misaligned(dout, dtype) || row_misaligned(y, dtype) || row_misaligned(dy, dtype) ||
      row_misaligned(weight, w_dtype) || row_misaligned(dweight, w_dtype) || (((uintptr_t)source | (uintptr_t)place) & 3u))
    return APEXW_ERR_ALIGN;
  TokenArgs a = token_args(tokens, k, width, dtype, source, place);
  a.x = dout, a.x_stride = dout_stride, a.y = y, a.y_stride = y_stride, a.weight = weight, a.out = dy, a.dweight = dweight;
  const int st = by_types(dtype, w_dtype, [&](auto d, auto w) {
    if (tokens > 0 && (dy || dweight))
      hipLaunchKernelGGL((combine_backward_kernel<decltype(d)::value, decltype(w)::value>), token_grid(a), dim3(kWG), 0,
                         (hipStream_t)stream, a);
  });
  return st ? st : launched();
}

extern "C" int apexw_embedding_forward(const void* ids, int32_t id_bytes, int64_t n, const void* weight, int64_t w_stride,
                                       int64_t vocab, int64_t width, int32_t dtype, float scale, void* out, void* stream) {
  if (!rows_ok(n, width) || vocab <= 0 || vocab > INT32_MAX - 1 || w_stride < 0 || (id_bytes != 4 && id_bytes != 8))
    return APEXW_ERR_ARG;
  if (n > 0 && (!ids || !weight || !out)) return APEXW_ERR_ARG;
  if (row_misaligned(weight, dtype) || row_misaligned(out, dtype) || ((uintptr_t)ids & (id_bytes - 1))) return APEXW_ERR_ALIGN;
  EmbeddingArgs a{};
  a.ids = ids, a.wide = id_bytes == 8, a.n = n, a.w = weight, a.stride = w_stride, a.vocab = (uint32_t)vocab;
  a.width = (int32_t)width, a.scale = scale, a.out = out, a.log_t = log_threads(width, dtype, true);
  const int64_t per = kWG >> a.log_t;
  const bool ok = by_row_type(dtype, [&](auto d) {
    if (n > 0)
      hipLaunchKernelGGL(embedding_kernel<decltype(d)::value>, groups_grid((n + per - 1) / per), dim3(kWG), 0, (hipStream_t)stream, a);
  });
  return ok ? launched() : APEXW_ERR_DTYPE;
}

extern "C" int64_t apexw_embedding_weight_grad_workspace(int64_t n, int64_t vocab, int64_t width) {
  if (!rows_ok(n, width) || vocab <= 0 || vocab > INT32_MAX - 1) return -APEXW_ERR_ARG;
  if (vocab > kMostWords) return -APEXW_ERR_SIZE;
  return GradPlan(nullptr, 4, n, (uint32_t)vocab, width).bytes;
}

extern "C" int apexw_embedding_weight_grad(const void* dy, int64_t dy_stride, const void* ids, int32_t id_bytes, int64_t n,
                                           int64_t vocab, int64_t width, int32_t dtype, float scale, void* dw,
                                           int32_t dw_dtype, void* workspace, void* stream) {
  if (!rows_ok(n, width) || vocab <= 0 || vocab > INT32_MAX - 1 || dy_stride < 0 || (id_bytes != 4 && id_bytes != 8))
    return APEXW_ERR_ARG;
  if (!dw || (n > 0 && (!dy || !ids || !workspace))) return APEXW_ERR_ARG;
  if (row_misaligned(dy, dtype) || row_misaligned(dw, dw_dtype) || ((uintptr_t)ids & (id_bytes - 1)) ||
      ((uintptr_t)workspace & 15u))
    return APEXW_ERR_ALIGN;
  if (vocab > kMostWords) return APEXW_ERR_SIZE;
  const GradPlan plan(ids, id_bytes, n, (uint32_t)vocab, width);
  hipStream_t s = (hipStream_t)stream;
  char* ws = (char*)workspace;
  EmbeddingArgs a{};
  a.n = n, a.w = dy, a.stride = dy_stride, a.vocab = (uint32_t)vocab, a.width = (int32_t)width, a.scale = scale, a.out = dw;
  a.log_block = plan.log_block;
  a.log_t = log_threads(width, dtype, false);
  a.many = (int32_t*)(ws + plan.space.bytes), a.ranges = (int32_t*)(ws + plan.space.bytes + plan.many);
  a.blocks = (float*)(ws + plan.space.bytes + plan.many + plan.ranges);
  const bool few = n <= kFewTokens;
  SortArgs sort = plan.sort;
  sort.clear = (char*)a.many, sort.clears = plan.many + plan.ranges;
  if (few) sort.clear = (char*)dw, sort.clears = vocab * width * (dw_dtype == APEXW_F32 ? 4 : 2);
  // rows a workgroup: 2048 workgroups and more, of up to 64 rows
  const int rows = (int)(vocab < 4096 ? 1 : vocab / 2048 < 64 ? vocab / 2048 : 64);
  const unsigned groups = (unsigned)((vocab + rows - 1) / rows);
  const int st = by_types(dtype, dw_dtype, [&](auto d, auto o) {
    constexpr int DT = decltype(d)::value, OD = decltype(o)::value;
    if (n <= kSmall) {
      a.sorted = sort.to = (u32x2*)ws;
      const int64_t clears = (sort.clears + kClear - 1) / kClear;
      const dim3 grid((unsigned)(1 + (clears < kClears ? clears : kClears)));
      if (n <= kFew * kSortThreads) hipLaunchKernelGGL(embedding_sort_kernel<kFew>, grid, dim3(kSortThreads), 0, s, sort);
      else hipLaunchKernelGGL(embedding_sort_kernel<kMost>, grid, dim3(kSortThreads), 0, s, sort);
    } else {
      a.sorted = launch_sort<false>(sort, plan.space, true, ws, s);
    }
    if (few) {
      const dim3 grid((unsigned)n, (unsigned)((width + 64 * kVec<DT> - 1) / (64 * kVec<DT>)));
      if (n > 0) hipLaunchKernelGGL((embedding_few_kernel<DT, OD>), grid, dim3(kWG), 0, s, a);
      return;
    }
    const int chunks = (int)((width + kVec<DT> - 1) / kVec<DT>);
    const unsigned blocks = (unsigned)((n + (1 << a.log_block) - 1) >> a.log_block);
    hipLaunchKernelGGL(embedding_blocks_kernel<DT>, dim3(blocks, (unsigned)((chunks + 63) / 64)), dim3(kWG), 0, s, a);
    hipLaunchKernelGGL((embedding_grad_kernel<DT, OD>), dim3(groups + kManyGroups), dim3(kWG), 0, s, a, rows);
  });
  return st ? st : launched();
}
