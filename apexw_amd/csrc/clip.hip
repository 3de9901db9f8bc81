// Global norm of a list of gradients, and their clipped copies (gfx950).
//
//   norm = (sum |g|^p)^(1/p) over every element of every tensor, p = 1, 2 or infinity
//   c = min(max_norm / (norm + 1e-6), 1), out = round(c g)
//
// Bound by memory: the norm reads every gradient, the scaling reads them again and writes the copies.
// Measured: 872 M fp32 gradients clipped to bf16 591 + 1027 us, 5.9 and 5.1 TB/s; 204 M in 2000 ragged bf16
// tensors 115 + 145 us (the norm 77, 5.3 TB/s, unless the copies of a call just before are still on their way out
// of the cache; one tensor of that size 109 or 71 + 142); a 6-tensor MLP 4.5 + 3.9 us.  The norm has to be known before the
// first element is written, so the gradients are read twice where they exceed the 256 MB cache; the scaling
// starts with what the norm's pass read last.
// Two launches.  The first leaves one partial sum per workgroup; every workgroup of the second adds the
// partials up in the same order, so all use one coefficient bit for bit, and nothing is atomic or cleared
// beforehand.
#include "common.h"

namespace {

constexpr int kUnit = APEXW_CLIP_UNIT;   // elements of a work unit: 32 per thread

struct __attribute__((packed, aligned(2))) Bytes16 { u32x4 v; };

// 8 elements from element e of a tensor, those below cnt (the rest 0): no alignment beyond the element's
template <int DT> APEXW_DEV void load_some(const void* base, int64_t e, int64_t cnt, float (&x)[8]) {
  if (cnt >= 8) {
    if constexpr (DT == APEXW_F32) {
      const auto p = APEXW_GLOBAL(const Bytes16, (const float*)base + e);
      const u32x4 a = p[0].v, b = p[1].v;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[j] = __uint_as_float(a[j]);
        x[4 + j] = __uint_as_float(b[j]);
      }
    } else {
      const u32x4 a = APEXW_GLOBAL(const Bytes16, (const uint16_t*)base + e)->v;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (DT == APEXW_BF16) {
          x[2 * j] = __uint_as_float(a[j] << 16);
          x[2 * j + 1] = __uint_as_float(a[j] & 0xFFFF0000u);
        } else {
          x[2 * j] = f16_bits_to_f32(a[j] & 0xFFFFu);
          x[2 * j + 1] = f16_bits_to_f32(a[j] >> 16);
        }
      }
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = j < cnt ? load1<DT>(base, e + j) : 0.0f;
}

template <int DT> APEXW_DEV void store_some(void* base, int64_t e, int64_t cnt, const float (&x)[8]) {
  uint32_t w[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (DT == APEXW_BF16) w[j] = pack_bf16x2(x[2 * j], x[2 * j + 1]);
    else if constexpr (DT == APEXW_F16) w[j] = f32_to_f16_bits(x[2 * j]) | (f32_to_f16_bits(x[2 * j + 1]) << 16);
  }
  if (cnt >= 8) {
    if constexpr (DT == APEXW_F32) {
      auto p = APEXW_GLOBAL(Bytes16, (float*)base + e);
      p[0].v = u32x4{__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])};
      p[1].v = u32x4{__float_as_uint(x[4]), __float_as_uint(x[5]), __float_as_uint(x[6]), __float_as_uint(x[7])};
    } else {
      APEXW_GLOBAL(Bytes16, (uint16_t*)base + e)->v = u32x4{w[0], w[1], w[2], w[3]};
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < cnt) {
      if constexpr (DT == APEXW_F32) APEXW_GLOBAL(float, base)[e + j] = x[j];
      else APEXW_GLOBAL(uint16_t, base)[e + j] = (uint16_t)(w[j >> 1] >> (16 * (j & 1)));
    }
}

// A list's table in device memory, or, a short list's, in the launch's own arguments: nothing to upload
struct Long {
  const apexw_clip_tensor* t;
};
struct Short {
  apexw_clip_tensor t[APEXW_CLIP_SMALL];
};

// the tensor of the table that holds unit u: the last one whose first unit is <= u (a tensor without
// elements has no units and the first unit of the next)
template <class Table> APEXW_DEV int find_tensor(const Table& tab, int n, int64_t u) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (tab.t[mid].first_unit <= u) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// the magnitudes of one thread's 32 elements of a unit joined into acc: sums of |x|^order (1, 2; a sum of
// squares that leaves the fp32 range is formed again in 64 bits, upwards by its infinity, downwards where it is
// so small that squares below the normal numbers may be part of it), or (order 0) the largest magnitude's bits,
// which order NaN above infinity above every number
template <int GD, int order> APEXW_DEV void unit_norm(const apexw_clip_tensor& t, int64_t e0, double& acc, uint32_t& top) {
  float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  uint32_t bits = 0u;   // of any element but zero
#pragma unroll
  for (int i = 0; i < kUnit / 2048; ++i) {
    const int64_t e = e0 + 2048 * i + 8 * threadIdx.x;
    float x[8];
    load_some<GD>(t.g, e, t.n - e, x);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if constexpr (order == 2) {
        s[j & 3] = fmaf(x[j], x[j], s[j & 3]);
        bits |= __float_as_uint(x[j]) << 1;
      } else if constexpr (order == 1) s[j & 3] += fabsf(x[j]);
      else {
        const uint32_t b = __float_as_uint(x[j]) & 0x7FFFFFFFu;
        top = b > top ? b : top;
      }
    }
  }
  if (order == 0) return;
  const float sum = (s[0] + s[1]) + (s[2] + s[3]);
  // 32 squares lose at most 2^-145 in all by underflow: nothing next to 2^-96
  if (__builtin_isinf(sum) || (order == 2 && sum < 0x1p-96f && bits != 0u)) {
    double d = 0.0;
    for (int i = 0; i < kUnit / 2048; ++i) {
      const int64_t e = e0 + 2048 * i + 8 * threadIdx.x;
      float x[8];
      load_some<GD>(t.g, e, t.n - e, x);
      for (int j = 0; j < 8; ++j) d += order == 2 ? (double)x[j] * x[j] : fabs((double)x[j]);
    }
    acc += d;
  } else {
    acc += (double)sum;
  }
}

APEXW_DEV double wave_sum_d(double x) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) x += __shfl_xor(x, off, 64);
  return x;
}
APEXW_DEV uint32_t wave_max_u(uint32_t x) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const uint32_t y = __shfl_xor(x, off, 64);
    x = y > x ? y : x;
  }
  return x;
}

// sum (or, order 0, the largest magnitude) over the workgroup's threads, on all of them
APEXW_DEV double join(double acc, uint32_t top, int order, double* red) {
  const double v = order == 0 ? (double)__uint_as_float(wave_max_u(top)) : wave_sum_d(acc);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  double s = red[0];
  for (int i = 1; i < 4; ++i) s = order != 0 ? s + red[i] : red[i] > s || red[i] != red[i] ? red[i] : s;
  __syncthreads();
  return s;
}

template <class Table, int order>
__global__ __launch_bounds__(256) void grad_norm_kernel(Table tab, int32_t n_tensors, int64_t n_units,
                                                        double* __restrict__ partial) {
  __shared__ double red[4];
  const int64_t u0 = n_units * blockIdx.x / gridDim.x, u1 = n_units * (blockIdx.x + 1) / gridDim.x;
  double acc = 0.0;
  uint32_t top = 0u;
  if (u0 < u1) {
    int k = find_tensor(tab, n_tensors, u0);
    apexw_clip_tensor t = tab.t[k];
    for (int64_t u = u0; u < u1; ++u) {
      while (u >= t.first_unit + (t.n + kUnit - 1) / kUnit) t = tab.t[++k];
      const int64_t e0 = (u - t.first_unit) * kUnit;
      if (t.g_dtype == APEXW_F32) unit_norm<APEXW_F32, order>(t, e0, acc, top);
      else if (t.g_dtype == APEXW_BF16) unit_norm<APEXW_BF16, order>(t, e0, acc, top);
      else unit_norm<APEXW_F16, order>(t, e0, acc, top);
    }
  }
  const double s = join(acc, top, order, red);
  if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

// the norm from the first launch's partials, in one order for every workgroup
APEXW_DEV float total_norm(const double* __restrict__ partial, int32_t n_partial, int32_t order, double* red) {
  double acc = 0.0;
  float top = 0.0f;
  for (int i = threadIdx.x; i < n_partial; i += 256) {
    if (order != 0) acc += partial[i];
    else {
      const float v = (float)partial[i];
      top = __float_as_uint(v) > __float_as_uint(top) ? v : top;
    }
  }
  const double s = join(acc, __float_as_uint(top), order, red);
  return (float)(order == 2 ? sqrt(s) : s);
}

__global__ __launch_bounds__(256) void total_norm_kernel(const double* __restrict__ partial, int32_t n_partial,
                                                         int32_t order, float* __restrict__ norm) {
  __shared__ double red[4];
  const float v = total_norm(partial, n_partial, order, red);
  if (threadIdx.x == 0) *norm = v;
}

template <int GD, int OD> APEXW_DEV void unit_scale(const apexw_clip_tensor& t, int64_t e0, float c) {
#pragma unroll
  for (int i = 0; i < kUnit / 2048; ++i) {
    const int64_t e = e0 + 2048 * i + 8 * threadIdx.x;
    if (e >= t.n) break;
    float x[8];
    load_some<GD>(t.g, e, t.n - e, x);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] *= c;
    store_some<OD>(t.out, e, t.n - e, x);
  }
}

template <int GD> APEXW_DEV void unit_scale_to(const apexw_clip_tensor& t, int64_t e0, float c) {
  if (t.out_dtype == APEXW_F32) unit_scale<GD, APEXW_F32>(t, e0, c);
  else if (t.out_dtype == APEXW_BF16) unit_scale<GD, APEXW_BF16>(t, e0, c);
  else unit_scale<GD, APEXW_F16>(t, e0, c);
}

// given: a norm that the caller formed (over more than these tensors); else the partials' norm, written to *norm.
// A tensor clipped in place is left alone where the coefficient is one.
template <class Table>
__global__ __launch_bounds__(256) void grad_scale_kernel(Table tab, int32_t n_tensors,
                                                         int64_t n_units, int32_t order,
                                                         const double* __restrict__ partial, int32_t n_partial,
                                                         const float* __restrict__ given, float max_norm,
                                                         float* __restrict__ norm) {
  __shared__ double red[4];
  const float total = given ? *given : total_norm(partial, n_partial, order, red);
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = total;
  const float q = max_norm / (total + 1e-6f), c = q > 1.0f ? 1.0f : q;   // NaN stays NaN
  // the last units first: what the norm's pass read last is still in the cache
  const int64_t b = gridDim.x - 1 - blockIdx.x;
  const int64_t u0 = n_units * b / gridDim.x, u1 = n_units * (b + 1) / gridDim.x;
  if (u0 >= u1) return;
  int k = find_tensor(tab, n_tensors, u1 - 1);
  apexw_clip_tensor t = tab.t[k];
  for (int64_t u = u1 - 1; u >= u0; --u) {
    while (u < t.first_unit) t = tab.t[--k];
    if (c == 1.0f && t.out == t.g) continue;
    const int64_t e0 = (u - t.first_unit) * kUnit;
    if (t.g_dtype == APEXW_F32) unit_scale_to<APEXW_F32>(t, e0, c);
    else if (t.g_dtype == APEXW_BF16) unit_scale_to<APEXW_BF16>(t, e0, c);
    else unit_scale_to<APEXW_F16>(t, e0, c);
  }
}

// entries from the launch's arguments into a table on the device
__global__ __launch_bounds__(64) void clip_upload_kernel(Short tab, int32_t n, apexw_clip_tensor* __restrict__ to) {
  if ((int)threadIdx.x < n) to[threadIdx.x] = tab.t[threadIdx.x];
}

int norm_grid(int64_t n_units) { return (int)(n_units < APEXW_CLIP_PARTIALS ? (n_units > 0 ? n_units : 1) : APEXW_CLIP_PARTIALS); }

bool table_ok(const apexw_clip_tensor* tensors, int32_t n_tensors, int64_t n_units) {
  return n_tensors >= 0 && n_units >= 0 && (n_units == 0 || (tensors && n_tensors > 0 && !((uintptr_t)tensors & 7u)));
}
bool order_ok(int32_t order) { return order >= 0 && order <= 2; }
bool max_ok(float m) { return m >= 0.0f; }

}  // namespace

extern "C" int64_t apexw_clip_layout(apexw_clip_tensor* t, int32_t n_tensors) {
  if (n_tensors < 0 || (n_tensors > 0 && !t)) return -APEXW_ERR_ARG;
  int64_t units = 0;
  for (int32_t i = 0; i < n_tensors; ++i) {
    if (t[i].n < 0 || (t[i].n > 0 && !t[i].g)) return -APEXW_ERR_ARG;
    if (t[i].g_dtype > APEXW_F16 || t[i].out_dtype > APEXW_F16) return -APEXW_ERR_DTYPE;
    if (((uintptr_t)t[i].g & (t[i].g_dtype == APEXW_F32 ? 3u : 1u)) ||
        ((uintptr_t)t[i].out & (t[i].out_dtype == APEXW_F32 ? 3u : 1u)))
      return -APEXW_ERR_ALIGN;
    t[i].first_unit = units;
    units += (t[i].n + kUnit - 1) / kUnit;
  }
  return units;
}

extern "C" int apexw_clip_upload(const apexw_clip_tensor* host, int32_t n_tensors, apexw_clip_tensor* device, void* stream) {
  if (n_tensors < 0 || (n_tensors > 0 && (!host || !device))) return APEXW_ERR_ARG;
  if ((uintptr_t)device & 7u) return APEXW_ERR_ALIGN;
  if (n_tensors == 0) return APEXW_OK;
  static_assert(APEXW_CLIP_SMALL <= 64, "a thread an entry");
  for (int32_t i = 0; i < n_tensors; i += APEXW_CLIP_SMALL) {
    const int32_t n = n_tensors - i < APEXW_CLIP_SMALL ? n_tensors - i : APEXW_CLIP_SMALL;
    Short tab{};
    for (int32_t j = 0; j < n; ++j) tab.t[j] = host[i + j];
    hipLaunchKernelGGL(clip_upload_kernel, dim3(1), dim3(64), 0, (hipStream_t)stream, tab, n, device + i);
  }
  return hipGetLastError() == hipSuccess ? APEXW_OK : APEXW_ERR_LAUNCH;
}

namespace {

template <class Table>
void norm_partials(const Table& tab, int32_t n_tensors, int64_t n_units, int32_t order, double* workspace, int grid,
                   hipStream_t stream) {
  if (order == 2)
    hipLaunchKernelGGL((grad_norm_kernel<Table, 2>), dim3(grid), dim3(256), 0, stream, tab, n_tensors, n_units, workspace);
  else if (order == 1)
    hipLaunchKernelGGL((grad_norm_kernel<Table, 1>), dim3(grid), dim3(256), 0, stream, tab, n_tensors, n_units, workspace);
  else
    hipLaunchKernelGGL((grad_norm_kernel<Table, 0>), dim3(grid), dim3(256), 0, stream, tab, n_tensors, n_units, workspace);
}

template <class Table>
int clip(const Table& tab, int32_t n_tensors, int64_t n_units, int32_t order, float max_norm, double* workspace,
         float* norm, hipStream_t stream) {
  const int grid = norm_grid(n_units);
  norm_partials(tab, n_tensors, n_units, order, workspace, grid, stream);
  hipLaunchKernelGGL(grad_scale_kernel<Table>, dim3(grid), dim3(256), 0, stream, tab, n_tensors, n_units, order,
                     workspace, grid, (const float*)nullptr, max_norm, norm);
  return hipGetLastError() == hipSuccess ? APEXW_OK : APEXW_ERR_LAUNCH;
}

}  // namespace

extern "C" int apexw_grad_norm(const apexw_clip_tensor* tensors, int32_t n_tensors, int64_t n_units, int32_t order,
                               double* workspace, float* norm, void* stream) {
  if (!table_ok(tensors, n_tensors, n_units) || !order_ok(order) || !workspace || !norm) return APEXW_ERR_ARG;
  const int grid = norm_grid(n_units);
  norm_partials(Long{tensors}, n_tensors, n_units, order, workspace, grid, (hipStream_t)stream);
  hipLaunchKernelGGL(total_norm_kernel, dim3(1), dim3(256), 0, (hipStream_t)stream, workspace, grid, order, norm);
  return hipGetLastError() == hipSuccess ? APEXW_OK : APEXW_ERR_LAUNCH;
}

extern "C" int apexw_grad_scale(const apexw_clip_tensor* tensors, int32_t n_tensors, int64_t n_units,
                                const float* norm, float max_norm, void* stream) {
  if (!table_ok(tensors, n_tensors, n_units) || !norm || !max_ok(max_norm)) return APEXW_ERR_ARG;
  if (n_units == 0) return APEXW_OK;
  hipLaunchKernelGGL(grad_scale_kernel<Long>, dim3(norm_grid(n_units)), dim3(256), 0, (hipStream_t)stream,
                     Long{tensors}, n_tensors, n_units, 2, (const double*)nullptr, 0, norm, max_norm, (float*)nullptr);
  return hipGetLastError() == hipSuccess ? APEXW_OK : APEXW_ERR_LAUNCH;
}

extern "C" int apexw_clip_grads(const apexw_clip_tensor* tensors, int32_t n_tensors, int64_t n_units, int32_t order,
                                float max_norm, double* workspace, float* norm, void* stream) {
  if (!table_ok(tensors, n_tensors, n_units) || !order_ok(order) || !max_ok(max_norm) || !workspace || !norm)
    return APEXW_ERR_ARG;
  return clip(Long{tensors}, n_tensors, n_units, order, max_norm, workspace, norm, (hipStream_t)stream);
}

extern "C" int apexw_clip_grads_small(const apexw_clip_tensor* tensors, int32_t n_tensors, int64_t n_units, int32_t order,
                                      float max_norm, double* workspace, float* norm, void* stream) {
  if (!table_ok(tensors, n_tensors, n_units) || !order_ok(order) || !max_ok(max_norm) || !workspace || !norm)
    return APEXW_ERR_ARG;
  if (n_tensors > APEXW_CLIP_SMALL) return APEXW_ERR_SIZE;
  Short tab{};
  for (int32_t i = 0; i < n_tensors; ++i) tab.t[i] = tensors[i];
  return clip(tab, n_tensors, n_units, order, max_norm, workspace, norm, (hipStream_t)stream);
}
