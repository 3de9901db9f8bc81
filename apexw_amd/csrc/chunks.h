// Rows as chunks of 16 bytes at any element address (gfx950): global accesses need no alignment, so a row of odd width
// starts anywhere, and its last chunk is taken from its end, over elements that the one before has too.
#pragma once

#include "common.h"

namespace {

template <int DT> constexpr int kVec = DT == APEXW_F32 ? 4 : 8;   // elements of a chunk

struct __attribute__((packed, aligned(2))) Chunk2 { u32x4 v; };
struct __attribute__((packed, aligned(4))) Chunk4 { u32x4 v; };

template <int DT> APEXW_DEV u32x4 chunk_at(const void* base, int64_t e) {
  if constexpr (DT == APEXW_F32) return APEXW_GLOBAL(const Chunk4, (const float*)base + e)->v;
  else return APEXW_GLOBAL(const Chunk2, (const uint16_t*)base + e)->v;
}
template <int DT> APEXW_DEV void chunk_to(void* base, int64_t e, u32x4 w) {
  if constexpr (DT == APEXW_F32) APEXW_GLOBAL(Chunk4, (float*)base + e)->v = w;
  else APEXW_GLOBAL(Chunk2, (uint16_t*)base + e)->v = w;
}
// the first cnt (0 .. kVec) elements of a chunk, the rest 0
template <int DT> APEXW_DEV u32x4 part_at(const void* base, int64_t e, int cnt) {
  u32x4 r = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int j = 0; j < kVec<DT>; ++j)
    if (j < cnt) {
      if constexpr (DT == APEXW_F32) r[j] = APEXW_GLOBAL(const uint32_t, base)[e + j];
      else r[j >> 1] |= (uint32_t)APEXW_GLOBAL(const uint16_t, base)[e + j] << (16 * (j & 1));
    }
  return r;
}
template <int DT> APEXW_DEV void part_to(void* base, int64_t e, int cnt, u32x4 w) {
#pragma unroll
  for (int j = 0; j < kVec<DT>; ++j)
    if (j < cnt) {
      if constexpr (DT == APEXW_F32) APEXW_GLOBAL(uint32_t, base)[e + j] = w[j];
      else APEXW_GLOBAL(uint16_t, base)[e + j] = (uint16_t)(w[j >> 1] >> (16 * (j & 1)));
    }
}

// The chunks of a row of `width` elements: chunk c has the elements from begin(c) on, all kVec of them where the row is
// as long as a chunk; skip(c): how many of them the chunk before has too
template <int DT> struct RowChunks {
  int width, count;
  __device__ __forceinline__ explicit RowChunks(int w) : width(w), count((w + kVec<DT> - 1) / kVec<DT>) {}
  __device__ __forceinline__ int begin(int c) const {
    const int at = c * kVec<DT>, last = width - kVec<DT>;
    return at <= last ? at : last < 0 ? 0 : last;
  }
  __device__ __forceinline__ int skip(int c) const { return c * kVec<DT> - begin(c); }
  __device__ __forceinline__ u32x4 load(const void* row, int c) const {
    return width >= kVec<DT> ? chunk_at<DT>(row, begin(c)) : part_at<DT>(row, 0, width);
  }
  __device__ __forceinline__ void store(void* row, int c, u32x4 w) const {
    if (width >= kVec<DT>) chunk_to<DT>(row, begin(c), w);
    else part_to<DT>(row, 0, width, w);
  }
};

template <int DT> APEXW_DEV void values(u32x4 w, float (&x)[kVec<DT>]) {
#pragma unroll
  for (int j = 0; j < kVec<DT>; ++j) {
    if constexpr (DT == APEXW_F32) x[j] = __uint_as_float(w[j]);
    else if constexpr (DT == APEXW_BF16) x[j] = __uint_as_float(j & 1 ? w[j >> 1] & 0xFFFF0000u : w[j >> 1] << 16);
    else x[j] = f16_bits_to_f32(w[j >> 1] >> (16 * (j & 1)) & 0xFFFFu);
  }
}
// rounded to nearest even
template <int DT> APEXW_DEV u32x4 rounded(const float (&x)[kVec<DT>]) {
  u32x4 w;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    if constexpr (DT == APEXW_F32) w[q] = __float_as_uint(x[q]);
    else if constexpr (DT == APEXW_BF16) w[q] = pack_bf16x2(x[2 * q], x[2 * q + 1]);
    else w[q] = f32_to_f16_bits(x[2 * q]) | f32_to_f16_bits(x[2 * q + 1]) << 16;
  }
  return w;
}
template <int DT> APEXW_DEV const void* row_at(const void* base, int64_t e) {
  return (const char*)base + e * Elem<DT>::bytes;
}
template <int DT> APEXW_DEV void* row_at(void* base, int64_t e) { return (char*)base + e * Elem<DT>::bytes; }

// f(the type code as a constant) for a type of rows; false for another code
template <class F> bool by_row_type(int32_t dtype, F&& f) {
  if (dtype == APEXW_F32) f(std::integral_constant<int, APEXW_F32>());
  else if (dtype == APEXW_BF16) f(std::integral_constant<int, APEXW_BF16>());
  else if (dtype == APEXW_F16) f(std::integral_constant<int, APEXW_F16>());
  else return false;
  return true;
}
inline bool row_misaligned(const void* p, int32_t dtype) { return ((uintptr_t)p & (dtype == APEXW_F32 ? 3u : 1u)) != 0; }

}  // namespace
