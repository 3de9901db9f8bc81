// Layer norm, forward and backward, with the reduction of the weight's and the bias's gradient (gfx950).
//
//   mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), xh = (x - mu) r, y = xh w + b
//   dx = r (g - mean(g) - xh mean(g xh)) with g = dy w;  dw = sum over rows of dy xh, db = of dy
//
// Both passes are bound by memory where rows are many: the forward reads x and writes y, the backward reads x
// and dy and writes dx.  A row is held in registers from its only read on, so its mean is taken before its squared
// deviations are summed (rows whose mean is far from zero lose nothing), all in fp32.
// Measured: forward 16384 x 4096 bf16 54 us, 4.95 TB/s (a copy of 4 GiB reaches 4.75); backward 16384 x 768 bf16
// with fp32 weights 19.0 us, 4.0 TB/s, and 3.9 for the columns (65536 rows 56.9 us, 5.3 TB/s); 4097 x 1021 fp32
// 13.6 and 4.6, 4096 x 1024 13.9 and 4.0; 8192 x 4096 fp32 88 us, 4.6 TB/s; one decode step's 8 x 768 3.7 us, most
// of it the launch.  Loading the next row before one is worked on cost more in registers than it hid (20.4 to
// 23.8 us).
// A chunk is 16 bytes of x; T threads share a row, NC chunks each.  Chunks may lie at any element
// address: a row of odd width starts anywhere, and global accesses need no alignment.
#include <type_traits>

#include "common.h"

namespace {

constexpr int kWG = 256;

template <int DT> constexpr int kVec = DT == APEXW_F32 ? 4 : 8;   // elements of a 16-byte chunk

struct __attribute__((packed, aligned(2))) Chunk16 { u32x4 v; };
struct __attribute__((packed, aligned(4))) Chunk32 { u32x4 v; };

// cnt (0 .. kVec) elements from element e of a row, the rest 0
template <int DT> APEXW_DEV u32x4 load_chunk(const void* base, int64_t e, int cnt) {
  constexpr int V = kVec<DT>;
  if (cnt >= V) {
    if constexpr (DT == APEXW_F32) return APEXW_GLOBAL(const Chunk32, (const float*)base + e)->v;
    else return APEXW_GLOBAL(const Chunk16, (const uint16_t*)base + e)->v;
  }
  u32x4 r = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int j = 0; j < V; ++j)
    if (j < cnt) {
      if constexpr (DT == APEXW_F32) r[j] = APEXW_GLOBAL(const uint32_t, base)[e + j];
      else r[j >> 1] |= (uint32_t)APEXW_GLOBAL(const uint16_t, base)[e + j] << (16 * (j & 1));
    }
  return r;
}

template <int DT> APEXW_DEV void store_chunk(void* base, int64_t e, int cnt, u32x4 w) {
  constexpr int V = kVec<DT>;
  if (cnt >= V) {
    if constexpr (DT == APEXW_F32) APEXW_GLOBAL(Chunk32, (float*)base + e)->v = w;
    else APEXW_GLOBAL(Chunk16, (uint16_t*)base + e)->v = w;
    return;
  }
#pragma unroll
  for (int j = 0; j < V; ++j)
    if (j < cnt) {
      if constexpr (DT == APEXW_F32) APEXW_GLOBAL(uint32_t, base)[e + j] = w[j];
      else APEXW_GLOBAL(uint16_t, base)[e + j] = (uint16_t)(w[j >> 1] >> (16 * (j & 1)));
    }
}

template <int DT> APEXW_DEV float chunk_get(u32x4 w, int j) {
  if constexpr (DT == APEXW_F32) return __uint_as_float(w[j]);
  else if constexpr (DT == APEXW_BF16)
    return (j & 1) ? __uint_as_float(w[j >> 1] & 0xFFFF0000u) : __uint_as_float(w[j >> 1] << 16);
  else return f16_bits_to_f32((w[j >> 1] >> (16 * (j & 1))) & 0xFFFFu);
}

// kVec values rounded to nearest even (fp16: overflow is infinity, as torch's conversion)
template <int DT, int V> APEXW_DEV u32x4 chunk_of(const float (&x)[V]) {
  u32x4 w;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (DT == APEXW_F32) w[j] = __float_as_uint(x[j]);
    else if constexpr (DT == APEXW_BF16) w[j] = pack_bf16x2(x[2 * j], x[2 * j + 1]);
    else w[j] = f32_to_f16_bits(x[2 * j]) | (f32_to_f16_bits(x[2 * j + 1]) << 16);
  }
  return w;
}

// V elements of the weight or the bias from element e, as fp32 (cnt of them, the rest 0)
template <int WD, int V> APEXW_DEV void load_param(const void* base, int64_t e, int cnt, float (&x)[V]) {
#pragma unroll
  for (int q = 0; q < V / kVec<WD>; ++q) {
    const u32x4 w = load_chunk<WD>(base, e + q * kVec<WD>, cnt - q * kVec<WD>);
#pragma unroll
    for (int j = 0; j < kVec<WD>; ++j) x[q * kVec<WD> + j] = chunk_get<WD>(w, j);
  }
}

template <int DT> APEXW_DEV void store_elem(void* base, int64_t i, float x) {
  if constexpr (DT == APEXW_F32) APEXW_GLOBAL(float, base)[i] = x;
  else if constexpr (DT == APEXW_BF16) APEXW_GLOBAL(uint16_t, base)[i] = (uint16_t)f32_to_bf16_bits(x);
  else APEXW_GLOBAL(uint16_t, base)[i] = (uint16_t)f32_to_f16_bits(x);
}

// Sum over T <= 64 lanes that stand together
template <int T> APEXW_DEV float lanes_sum(float x) {
#pragma unroll
  for (int off = T < 64 ? T / 2 : 32; off > 0; off >>= 1) x += __shfl_xor(x, off, 64);
  return x;
}
// Sum over the T threads of a row; red: T / 64 floats that nobody else uses until the next barrier
template <int T> APEXW_DEV float row_sum(float x, float* red) {
  x = lanes_sum<T>(x);
  if constexpr (T > 64) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
    __syncthreads();
    x = 0.0f;
#pragma unroll
    for (int i = 0; i < T / 64; ++i) x += red[i];
  }
  return x;
}

struct LnArgs {
  const void *x, *dy, *w, *b;
  int64_t x_stride, dy_stride, rows;
  void *y, *dw, *db;      // y: the output, or dx
  float *mean, *rstd, *partial;
  int32_t width;
  float eps, inv_width;
};

APEXW_DEV int clamp_cnt(int left, int most) { return left < 0 ? 0 : left < most ? left : most; }

// One row per T threads (T = 64: a wave each; narrow rows share one), rows r, r + grid's rows, ...; the weights stay in registers.
template <int XD, int WD, int T, int NC>
__global__ __launch_bounds__(T < kWG ? kWG : T) void ln_forward_kernel(LnArgs a) {
  constexpr int V = kVec<XD>, kRows = T < kWG ? kWG / T : 1;
  __shared__ float red[2][T > 64 ? T / 64 : 1];
  const int t = T < kWG ? threadIdx.x % T : threadIdx.x;
  int64_t row = (int64_t)blockIdx.x * kRows + (T < kWG ? threadIdx.x / T : 0);
  const int64_t step = (int64_t)gridDim.x * kRows;
  for (; row < a.rows; row += step) {
    const char* src = (const char*)a.x + row * a.x_stride * (int64_t)Elem<XD>::bytes;
    u32x4 raw[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int e = (t + T * i) * V;
      raw[i] = load_chunk<XD>(src, e, clamp_cnt(a.width - e, V));
    }
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) s += chunk_get<XD>(raw[i], j);
    const float mean = row_sum<T>(s, red[0]) * a.inv_width;
    float q = 0.0f;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      // what is missing was read as 0 and deviates by 0: from the mean taken as 0 where a whole chunk is
      const int cnt = clamp_cnt(a.width - (t + T * i) * V, V);
      const float mu = cnt > 0 ? mean : 0.0f;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float d = chunk_get<XD>(raw[i], j) - mu;
        if (cnt == V || cnt == 0 || j < cnt) q = fmaf(d, d, q);
      }
    }
    const float rstd = 1.0f / sqrtf(fmaf(row_sum<T>(q, red[1]), a.inv_width, a.eps));
    if (t == 0) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
    char* dst = (char*)a.y + row * a.width * (int64_t)Elem<XD>::bytes;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int e = (t + T * i) * V, cnt = clamp_cnt(a.width - e, V);
      if (cnt == 0) continue;
      float w[V], b[V], y[V];
#pragma unroll
      for (int j = 0; j < V; ++j) w[j] = 1.0f, b[j] = 0.0f;
      if (a.w) load_param<WD>(a.w, e, cnt, w);
      if (a.b) load_param<WD>(a.b, e, cnt, b);
#pragma unroll
      for (int j = 0; j < V; ++j) y[j] = fmaf((chunk_get<XD>(raw[i], j) - mean) * rstd, w[j], b[j]);
      store_chunk<XD>(dst, e, cnt, chunk_of<XD>(y));
    }
  }
}

// Rows too long for registers: a workgroup per row, which it reads three times (the second and third from L2);
// 2048 x 32768 fp32 162 us.
template <int XD, int WD>
__global__ __launch_bounds__(1024) void ln_forward_long_kernel(LnArgs a) {
  constexpr int V = kVec<XD>, T = 1024;
  __shared__ float red[2][T / 64];
  const int t = threadIdx.x;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const char* src = (const char*)a.x + row * a.x_stride * (int64_t)Elem<XD>::bytes;
    float s = 0.0f, q = 0.0f;
    for (int64_t e = t * V; e < a.width; e += T * V) {
      const u32x4 raw = load_chunk<XD>(src, e, (int)(a.width - e < V ? a.width - e : V));
#pragma unroll
      for (int j = 0; j < V; ++j) s += chunk_get<XD>(raw, j);
    }
    const float mean = row_sum<T>(s, red[0]) * a.inv_width;
    for (int64_t e = t * V; e < a.width; e += T * V) {
      const int cnt = (int)(a.width - e < V ? a.width - e : V);
      const u32x4 raw = load_chunk<XD>(src, e, cnt);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float d = j < cnt ? chunk_get<XD>(raw, j) - mean : 0.0f;
        q = fmaf(d, d, q);
      }
    }
    const float rstd = 1.0f / sqrtf(fmaf(row_sum<T>(q, red[1]), a.inv_width, a.eps));
    if (t == 0) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
    char* dst = (char*)a.y + row * a.width * (int64_t)Elem<XD>::bytes;
    for (int64_t e = t * V; e < a.width; e += T * V) {
      const int cnt = (int)(a.width - e < V ? a.width - e : V);
      const u32x4 raw = load_chunk<XD>(src, e, cnt);
      float w[V], b[V], y[V];
#pragma unroll
      for (int j = 0; j < V; ++j) w[j] = 1.0f, b[j] = 0.0f;
      if (a.w) load_param<WD>(a.w, e, cnt, w);
      if (a.b) load_param<WD>(a.b, e, cnt, b);
#pragma unroll
      for (int j = 0; j < V; ++j) y[j] = fmaf((chunk_get<XD>(raw, j) - mean) * rstd, w[j], b[j]);
      store_chunk<XD>(dst, e, cnt, chunk_of<XD>(y));
    }
  }
}

// dx of rows r, r + grid's rows, ...; each thread sums dw and db of its columns over them, a workgroup's
// row groups join in LDS, and its sums go to partial[blockIdx.x][2][width].
template <int XD, int WD, int T, int NC>
__global__ __launch_bounds__(T < kWG ? kWG : T) void ln_backward_kernel(LnArgs a) {
  constexpr int V = kVec<XD>, kThreads = T < kWG ? kWG : T, kRows = kThreads / T;
  __shared__ float red[2][2][T > 64 ? T / 64 : 1];
  __shared__ float join[kRows > 1 ? (kRows - 1) * T * V : 1];
  const int t = threadIdx.x % T, group = threadIdx.x / T;
  float dw[NC][V], db[NC][V];
#pragma unroll
  for (int i = 0; i < NC; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) dw[i][j] = db[i][j] = 0.0f;
  int parity = 0;
  for (int64_t row = (int64_t)blockIdx.x * kRows + group; row < a.rows; row += (int64_t)gridDim.x * kRows) {
    const char* xs = (const char*)a.x + row * a.x_stride * (int64_t)Elem<XD>::bytes;
    const char* ds = (const char*)a.dy + row * a.dy_stride * (int64_t)Elem<XD>::bytes;
    const float mu = a.mean[row], rs = a.rstd[row];
    u32x4 x[NC], dy[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int e = (t + T * i) * V, cnt = clamp_cnt(a.width - e, V);
      x[i] = load_chunk<XD>(xs, e, cnt);
      dy[i] = load_chunk<XD>(ds, e, cnt);
    }
    float w[NC][V], s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int e = (t + T * i) * V, cnt = clamp_cnt(a.width - e, V);
#pragma unroll
      for (int j = 0; j < V; ++j) w[i][j] = 1.0f;
      if (a.w) load_param<WD>(a.w, e, cnt, w[i]);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        // behind the row's end dy is 0, and so is every product with a finite xh
        const float xh = (chunk_get<XD>(x[i], j) - mu) * rs, d = chunk_get<XD>(dy[i], j), g = d * w[i][j];
        dw[i][j] = fmaf(d, xh, dw[i][j]);
        db[i][j] += d;
        s1 += g;
        s2 = fmaf(g, xh, s2);
      }
    }
    if (!a.y) continue;
    // a mean so large over so small a deviation that xh behind the row's end is not: its own elements alone
    if (__builtin_expect(s2 != s2, 0)) {
      s2 = 0.0f;
#pragma unroll
      for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j)
          if ((t + T * i) * V + j < a.width)
            s2 = fmaf(chunk_get<XD>(dy[i], j) * w[i][j], (chunk_get<XD>(x[i], j) - mu) * rs, s2);
    }
    s1 = lanes_sum<T>(s1);
    s2 = lanes_sum<T>(s2);
    if constexpr (T > 64) {
      if ((threadIdx.x & 63) == 0) {
        red[parity][0][t >> 6] = s1;
        red[parity][1][t >> 6] = s2;
      }
      __syncthreads();
      s1 = s2 = 0.0f;
#pragma unroll
      for (int i = 0; i < T / 64; ++i) {
        s1 += red[parity][0][i];
        s2 += red[parity][1][i];
      }
      parity ^= 1;
    }
    s1 *= a.inv_width;
    s2 *= a.inv_width;
    char* dst = (char*)a.y + row * a.width * (int64_t)Elem<XD>::bytes;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int e = (t + T * i) * V, cnt = clamp_cnt(a.width - e, V);
      if (cnt == 0) continue;
      float y[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float xh = (chunk_get<XD>(x[i], j) - mu) * rs;
        y[j] = rs * (chunk_get<XD>(dy[i], j) * w[i][j] - fmaf(xh, s2, s1));
      }
      store_chunk<XD>(dst, e, cnt, chunk_of<XD>(y));
    }
  }
  if (!a.partial) return;
  float* out = a.partial + (int64_t)blockIdx.x * 2 * a.width;
  for (int half = 0; half < 2; ++half) {
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      float s[V];
#pragma unroll
      for (int j = 0; j < V; ++j) s[j] = half ? db[i][j] : dw[i][j];
      if constexpr (kRows > 1) {
        __syncthreads();
        if (group > 0)
#pragma unroll
          for (int j = 0; j < V; ++j) join[((group - 1) * V + j) * T + t] = s[j];
        __syncthreads();
        if (group == 0)
#pragma unroll
          for (int q = 0; q < kRows - 1; ++q)
#pragma unroll
            for (int j = 0; j < V; ++j) s[j] += join[(q * V + j) * T + t];
      }
      const int e = (t + T * i) * V;
      if (group == 0)
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (e + j < a.width) out[(int64_t)half * a.width + e + j] = s[j];
    }
  }
}

// dx of rows too long for registers: a workgroup per row, read twice.  An element a load: 4096 x 32768 bf16 338 us
// (2.4 TB/s), and 158 for the columns below.
template <int XD, int WD>
__global__ __launch_bounds__(1024) void ln_backward_long_kernel(LnArgs a) {
  constexpr int T = 1024;
  __shared__ float red[2][T / 64];
  const int t = threadIdx.x;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const char* xs = (const char*)a.x + row * a.x_stride * (int64_t)Elem<XD>::bytes;
    const char* ds = (const char*)a.dy + row * a.dy_stride * (int64_t)Elem<XD>::bytes;
    const float mean = a.mean[row], rstd = a.rstd[row];
    float s1 = 0.0f, s2 = 0.0f;
    for (int64_t e = t; e < a.width; e += T) {
      const float xh = (load1<XD>(xs, e) - mean) * rstd;
      const float g = load1<XD>(ds, e) * (a.w ? load1<WD>(a.w, e) : 1.0f);
      s1 += g;
      s2 = fmaf(g, xh, s2);
    }
    s1 = row_sum<T>(s1, red[0]) * a.inv_width;
    s2 = row_sum<T>(s2, red[1]) * a.inv_width;
    char* dst = (char*)a.y + row * a.width * (int64_t)Elem<XD>::bytes;
    for (int64_t e = t; e < a.width; e += T) {
      const float xh = (load1<XD>(xs, e) - mean) * rstd;
      const float g = load1<XD>(ds, e) * (a.w ? load1<WD>(a.w, e) : 1.0f);
      store_elem<XD>(dst, e, rstd * (g - fmaf(xh, s2, s1)));
    }
    __syncthreads();
  }
}

// Column sums of rows too long for registers: 256 columns a workgroup, rows blockIdx.y, + gridDim.y, ...
template <int XD>
__global__ __launch_bounds__(kWG) void ln_columns_kernel(LnArgs a) {
  const int64_t e = (int64_t)blockIdx.x * kWG + threadIdx.x;
  if (e >= a.width) return;
  float dw = 0.0f, db = 0.0f;
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const float xh = (load1<XD>((const char*)a.x + row * a.x_stride * (int64_t)Elem<XD>::bytes, e) - a.mean[row]) *
                     a.rstd[row];
    const float d = load1<XD>((const char*)a.dy + row * a.dy_stride * (int64_t)Elem<XD>::bytes, e);
    dw = fmaf(d, xh, dw);
    db += d;
  }
  a.partial[(int64_t)blockIdx.y * 2 * a.width + e] = dw;
  a.partial[(int64_t)blockIdx.y * 2 * a.width + a.width + e] = db;
}

// dw (blockIdx.y 0) and db (1): 32 columns a workgroup, 32 threads to a column, in a fixed order.
template <int WD>
__global__ __launch_bounds__(1024) void ln_reduce_kernel(const float* __restrict__ partial, int32_t n, int32_t width,
                                                         void* dw, void* db) {
  __shared__ float red[32][33];
  void* out = blockIdx.y ? db : dw;
  if (!out) return;
  const int c = threadIdx.x & 31, g = threadIdx.x >> 5;
  const int64_t e = (int64_t)blockIdx.x * 32 + c;
  float q[8] = {};   // eight loads in flight
  if (e < width) {
    const float* p = partial + (int64_t)blockIdx.y * width + e;
    int i = g;
    for (; i + 224 < n; i += 256)
#pragma unroll
      for (int j = 0; j < 8; ++j) q[j] += p[(int64_t)(i + 32 * j) * 2 * width];
    for (; i < n; i += 32) q[0] += p[(int64_t)i * 2 * width];
  }
  float s = ((q[0] + q[1]) + (q[2] + q[3])) + ((q[4] + q[5]) + (q[6] + q[7]));
  red[g][c] = s;
  __syncthreads();
  if (g != 0 || e >= width) return;
  s = 0.0f;
#pragma unroll
  for (int i = 0; i < 32; ++i) s += red[i][c];
  store_elem<WD>(out, e, s);
}

// Workgroups of a backward pass, at most: each leaves 8 bytes of partial sums a column.  Measured with 256, 512
// and 1024 of them: 16384 x 768 bf16 (rows of a wave) 42 / 28 / 20 us, 8192 x 4096 fp32 (256 threads) 122 / 93 /
// 111 us, 4096 x 8192 bf16 (512 threads) 68 / 68 / 92 us, 2048 x 16384 bf16 (1024 threads) 68 / 93 / 146 us.
constexpr int kMaxGroups = 1024;
template <int T> constexpr int kGroups = T <= 64 ? kMaxGroups : T == 256 ? 512 : 256;

template <int XD, int WD, int T, int NC>
void forward_as(const LnArgs& a, hipStream_t stream) {
  constexpr int kRows = T < kWG ? kWG / T : 1, kThreads = T < kWG ? kWG : T;
  const int64_t want = (a.rows + kRows - 1) / kRows;
  const int grid = (int)(want < (1 << 20) ? want : 1 << 20);
  hipLaunchKernelGGL((ln_forward_kernel<XD, WD, T, NC>), dim3(grid), dim3(kThreads), 0, stream, a);
}

template <int XD, int WD>
void forward(const LnArgs& a, hipStream_t stream) {
  const int chunks = (int)(((int64_t)a.width + kVec<XD> - 1) / kVec<XD>);
  if (chunks <= 16) forward_as<XD, WD, 16, 1>(a, stream);
  else if (chunks <= 32) forward_as<XD, WD, 32, 1>(a, stream);
  else if (chunks <= 64) forward_as<XD, WD, 64, 1>(a, stream);
  else if (chunks <= 128) forward_as<XD, WD, 64, 2>(a, stream);
  else if (chunks <= 256) forward_as<XD, WD, 64, 4>(a, stream);
  else if (chunks <= 512) forward_as<XD, WD, 256, 2>(a, stream);
  else if (chunks <= 1024) forward_as<XD, WD, 256, 4>(a, stream);
  else if (chunks <= 2048) forward_as<XD, WD, 1024, 2>(a, stream);
  else if (chunks <= 4096) forward_as<XD, WD, 1024, 4>(a, stream);
  else
    hipLaunchKernelGGL((ln_forward_long_kernel<XD, WD>), dim3((unsigned)(a.rows < 65536 ? a.rows : 65536)), dim3(1024),
                       0, stream, a);
}

template <int XD, int WD, int T, int NC>
int backward_as(const LnArgs& a, hipStream_t stream) {
  constexpr int kThreads = T < kWG ? kWG : T, kRows = kThreads / T;
  const int64_t want = (a.rows + kRows - 1) / kRows;
  const int grid = (int)(want < kGroups<T> ? want : kGroups<T>);
  hipLaunchKernelGGL((ln_backward_kernel<XD, WD, T, NC>), dim3(grid), dim3(kThreads), 0, stream, a);
  return grid;
}

template <int XD, int WD>
int backward(const LnArgs& a, hipStream_t stream) {
  const int chunks = (int)(((int64_t)a.width + kVec<XD> - 1) / kVec<XD>);
  constexpr int C = 8 / kVec<XD>;   // chunks of 8 elements: up to 16 elements a thread
  if (chunks <= 16 * C) return backward_as<XD, WD, 16, C>(a, stream);
  if (chunks <= 32 * C) return backward_as<XD, WD, 32, C>(a, stream);
  if (chunks <= 64 * C) return backward_as<XD, WD, 64, C>(a, stream);
  if (chunks <= 128 * C) return backward_as<XD, WD, 64, 2 * C>(a, stream);
  if (chunks <= 512 * C) return backward_as<XD, WD, 256, 2 * C>(a, stream);
  if (chunks <= 1024 * C) return backward_as<XD, WD, 512, 2 * C>(a, stream);
  if (chunks <= 2048 * C) return backward_as<XD, WD, 1024, 2 * C>(a, stream);
  if (a.y)
    hipLaunchKernelGGL((ln_backward_long_kernel<XD, WD>), dim3((unsigned)(a.rows < 65536 ? a.rows : 65536)), dim3(1024),
                       0, stream, a);
  const int groups = (int)(a.rows < 64 ? a.rows : 64);
  if (a.partial)
    hipLaunchKernelGGL((ln_columns_kernel<XD>), dim3((a.width + kWG - 1) / kWG, groups), dim3(kWG), 0, stream, a);
  return groups;
}

// f(dtype of x, dtype of the weights) for the types that are supported
template <class F> int by_type(int32_t dtype, int32_t w_dtype, F&& f) {
  using std::integral_constant;
  typedef integral_constant<int, APEXW_F32> F32;
  typedef integral_constant<int, APEXW_BF16> BF16;
  typedef integral_constant<int, APEXW_F16> F16;
  if (dtype == APEXW_F32 && w_dtype == APEXW_F32) f(F32{}, F32{});
  else if (dtype == APEXW_BF16 && w_dtype == APEXW_BF16) f(BF16{}, BF16{});
  else if (dtype == APEXW_BF16 && w_dtype == APEXW_F32) f(BF16{}, F32{});
  else if (dtype == APEXW_F16 && w_dtype == APEXW_F16) f(F16{}, F16{});
  else if (dtype == APEXW_F16 && w_dtype == APEXW_F32) f(F16{}, F32{});
  else return APEXW_ERR_DTYPE;
  return APEXW_OK;
}

bool misaligned(const void* p, int32_t dtype) { return ((uintptr_t)p & (dtype == APEXW_F32 ? 3u : 1u)) != 0; }

}  // namespace

extern "C" int64_t apexw_layer_norm_workspace(int64_t rows, int64_t width) {
  if (rows < 0 || width <= 0 || width > INT32_MAX - 8192) return -APEXW_ERR_ARG;
  return (rows < kMaxGroups ? rows : kMaxGroups) * 2 * width;
}

extern "C" int apexw_layer_norm_forward(const void* x, int64_t rows, int64_t width, int64_t x_stride, int32_t dtype,
                                        const void* weight, const void* bias, int32_t w_dtype, float eps, void* y,
                                        float* mean, float* rstd, void* stream) {
  if (!x || !y || !mean || !rstd || rows < 0 || width <= 0 || width > INT32_MAX - 8192 || x_stride < 0 || !(eps >= 0.0f))
    return APEXW_ERR_ARG;
  if (misaligned(x, dtype) || misaligned(y, dtype) || misaligned(weight, w_dtype) || misaligned(bias, w_dtype) ||
      misaligned(mean, APEXW_F32) || misaligned(rstd, APEXW_F32))
    return APEXW_ERR_ALIGN;
  LnArgs a{};
  a.x = x, a.x_stride = x_stride, a.rows = rows, a.width = (int32_t)width, a.w = weight, a.b = bias, a.y = y;
  a.mean = mean, a.rstd = rstd, a.eps = eps, a.inv_width = 1.0f / (float)width;
  const int st = by_type(dtype, w_dtype, [&](auto xd, auto wd) {
    if (rows > 0) forward<decltype(xd)::value, decltype(wd)::value>(a, (hipStream_t)stream);
  });
  if (st != APEXW_OK) return st;
  return hipGetLastError() == hipSuccess ? APEXW_OK : APEXW_ERR_LAUNCH;
}

extern "C" int apexw_layer_norm_backward(const void* dy, int64_t dy_stride, const void* x, int64_t x_stride,
                                         const float* mean, const float* rstd, const void* weight, int64_t rows,
                                         int64_t width, int32_t dtype, int32_t w_dtype, void* dx, void* dw, void* db,
                                         float* workspace, void* stream) {
  if (!dy || !x || !mean || !rstd || rows < 0 || width <= 0 || width > INT32_MAX - 8192 || x_stride < 0 || dy_stride < 0)
    return APEXW_ERR_ARG;
  if ((dw || db) && !workspace) return APEXW_ERR_ARG;
  if (misaligned(x, dtype) || misaligned(dy, dtype) || misaligned(dx, dtype) || misaligned(weight, w_dtype) ||
      misaligned(dw, w_dtype) || misaligned(db, w_dtype) || misaligned(mean, APEXW_F32) ||
      misaligned(rstd, APEXW_F32) || misaligned(workspace, APEXW_F32))
    return APEXW_ERR_ALIGN;
  LnArgs a{};
  a.x = x, a.x_stride = x_stride, a.dy = dy, a.dy_stride = dy_stride, a.rows = rows, a.width = (int32_t)width;
  a.w = weight, a.y = dx, a.dw = dw, a.db = db, a.mean = (float*)mean, a.rstd = (float*)rstd;
  a.partial = dw || db ? workspace : nullptr, a.inv_width = 1.0f / (float)width;
  const int st = by_type(dtype, w_dtype, [&](auto xd, auto wd) {
    constexpr int XD = decltype(xd)::value, WD = decltype(wd)::value;
    const int n = rows > 0 ? backward<XD, WD>(a, (hipStream_t)stream) : 0;
    if (a.partial)
      hipLaunchKernelGGL((ln_reduce_kernel<WD>), dim3((unsigned)((width + 31) / 32), 2), dim3(1024), 0,
                         (hipStream_t)stream, workspace, n, (int32_t)width, dw, db);
  });
  if (st != APEXW_OK) return st;
  return hipGetLastError() == hipSuccess ? APEXW_OK : APEXW_ERR_LAUNCH;
}
