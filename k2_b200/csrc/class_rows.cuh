// Rows of class scores as the kernels of token_scores.cu and distillation.cu read them.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/k2b200.h"
#include "common.cuh"

namespace k2b {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// What a kernel needs of k2b200_class_rows.
template <typename T>
struct Rows {
  const T *scores;
  int32_t classes;
  int64_t inner, outer_stride, inner_stride;
  const void *lengths;
  int32_t lengths_64;
};

struct RowPlace {
  int64_t o, i;
  bool counts;
};

// An element of an array of int32 or int64, as int64.
__device__ __forceinline__ int64_t IntAt(const void *ints, int32_t is_64, int64_t k) {
  return is_64 ? static_cast<const int64_t *>(ints)[k]
               : (int64_t)static_cast<const int32_t *>(ints)[k];
}

template <typename T>
__device__ __forceinline__ RowPlace PlaceOf(const Rows<T> &rows, int32_t r) {
  RowPlace p;
  const uint32_t inner = (uint32_t)rows.inner, o = (uint32_t)r / inner;
  p.o = o;
  p.i = (uint32_t)r - o * inner;
  p.counts = rows.lengths == nullptr || p.i < IntAt(rows.lengths, rows.lengths_64, p.o);
  return p;
}

__device__ __forceinline__ float ToFloat(float v) { return v; }
__device__ __forceinline__ float ToFloat(__half v) { return __half2float(v); }
__device__ __forceinline__ float ToFloat(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T FromFloat(float v);
template <>
__device__ __forceinline__ float FromFloat<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half FromFloat<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 FromFloat<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// 2^x, off by at most 2 units of the last place and 0 below 2^-126.
__device__ __forceinline__ float Exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Order of scores: an unsigned number that grows with the score, 0 for none.  NaN comes before all
// numbers and -0 equals +0.  With the class below it, two keys of a row are never equal.
__device__ __forceinline__ uint32_t OrderOf(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  if (v != v) return 0xffffffffu;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t KeyOf(float v, int32_t c) {
  return (uint64_t)OrderOf(v) << 32 | (uint32_t)~c;
}

__device__ __forceinline__ float TeamMax(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
  return v;
}
__device__ __forceinline__ float TeamSum(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}
__device__ __forceinline__ uint64_t TeamMax(uint64_t v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    const uint64_t o = __shfl_xor_sync(0xffffffffu, v, d);
    v = o > v ? o : v;
  }
  return v;
}

// A row's scores are turned into p_c = 2^((x_c - high) * scale) / sum: high the largest (0 where
// all are -inf), sum 0 where all are -inf.
struct RowNorm {
  float high, sum;
};

// What the entry points ask of a k2b200_class_rows.
static inline int32_t CheckRows(const k2b200_class_rows *rows) {
  K2B_REQUIRE(rows != nullptr, "NULL pointer");
  K2B_REQUIRE(rows->type >= K2B200_F32 && rows->type <= K2B200_BF16, "unknown type %d",
              rows->type);
  K2B_REQUIRE(rows->num_classes > 0, "rows of no class");
  K2B_REQUIRE(rows->outer >= 0 && rows->inner >= 0 && rows->outer < ((int64_t)1 << 31) &&
                  rows->inner < ((int64_t)1 << 31) &&
                  rows->outer * rows->inner < ((int64_t)1 << 31),
              "%lld x %lld rows are more than fit", (long long)rows->outer,
              (long long)rows->inner);
  K2B_REQUIRE(rows->scores != nullptr || rows->outer * rows->inner == 0, "NULL pointer");
  return kOk;
}

template <typename T>
static inline Rows<T> RowsOf(const k2b200_class_rows *rows) {
  Rows<T> r;
  r.scores = static_cast<const T *>(rows->scores);
  r.classes = rows->num_classes;
  r.inner = rows->inner;
  r.outer_stride = rows->outer_stride;
  r.inner_stride = rows->inner_stride;
  r.lengths = rows->lengths;
  r.lengths_64 = rows->lengths_64;
  return r;
}

}  // namespace k2b
