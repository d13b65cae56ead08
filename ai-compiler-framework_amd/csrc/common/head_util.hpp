// Shared by the 8-bit and vocabulary-head ops: views of row-major matrices
// whose rows may be any distance apart, and loads and stores of 8 consecutive
// elements at any element alignment (gfx950 takes unaligned vector accesses to
// global memory).
#pragma once

#include "hip_util.hpp"

namespace aicf::hip {

enum ElemKind { EL_F32 = 0, EL_F16 = 1, EL_BF16 = 2 };

inline bool elem_kind(const TensorDesc& t, int* k) {
  switch (dt(t)) {
    case DType::kF32: *k = EL_F32; return true;
    case DType::kF16: *k = EL_F16; return true;
    case DType::kBF16: *k = EL_BF16; return true;
    default: return false;
  }
}
inline bool is_fp8(const TensorDesc& t) { return dt(t) == DType::kF8E4M3 || dt(t) == DType::kF8E5M2; }

// Row stride of a [rows, cols] matrix with unit column stride; rows of an
// output lie apart, rows of an input may repeat (a broadcast view).
inline bool matrix_ld(const TensorDesc& t, bool output, int64_t* ld) {
  if (t.rank != 2 || t.shape[0] < 0 || t.shape[1] < 0) return false;
  if (t.shape[1] > 1 && t.stride[1] != 1) return false;
  *ld = t.shape[0] > 1 ? t.stride[0] : t.shape[1];
  if (*ld < 0) return false;
  return !output || t.shape[0] <= 1 || *ld >= t.shape[1];
}
inline bool vector_of(const TensorDesc& t, DType d, int64_t n) {
  return dt(t) == d && t.rank == 1 && t.shape[0] == n && (n <= 1 || t.stride[0] == 1);
}
inline bool no_memory(const TensorDesc& t) { return !t.data && numel_of(t) > 0; }

// Whether any output meets an input or another output.
inline bool any_overlap(const TensorDesc* in, int ni, const TensorDesc* out, int no) {
  for (int i = 0; i < no; ++i) {
    for (int j = 0; j < ni; ++j)
      if (views_overlap(out[i], in[j])) return true;
    for (int j = 0; j < i; ++j)
      if (views_overlap(out[i], out[j])) return true;
  }
  return false;
}

// ---- 8 consecutive elements ------------------------------------------------
typedef float f32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint16_t u16x8_a2 __attribute__((ext_vector_type(8), aligned(2)));
typedef uint32_t u32x2_a1 __attribute__((ext_vector_type(2), aligned(1)));
typedef uint32_t u32x4_a1 __attribute__((ext_vector_type(4), aligned(1)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

template <int EK>
__device__ __forceinline__ float elem_f32(const void* p, int64_t i) {
  if constexpr (EK == EL_F32) return static_cast<const float*>(p)[i];
  const uint16_t h = static_cast<const uint16_t*>(p)[i];
  return EK == EL_F16 ? f16_to_f32(h) : bf16_to_f32(h);
}

// v[e] = p[i + e] for e < n, 0 behind (n may be anything).
template <int EK>
__device__ __forceinline__ void load8(float (&v)[8], const void* p, int64_t i, int64_t n) {
  if (n >= 8) {
    if constexpr (EK == EL_F32) {
      const float* q = static_cast<const float*>(p) + i;
      const f32x4_a4 a = *reinterpret_cast<const f32x4_a4*>(q), b = *reinterpret_cast<const f32x4_a4*>(q + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] = a[e];
        v[4 + e] = b[e];
      }
    } else {
      const u16x8_a2 a = *reinterpret_cast<const u16x8_a2*>(static_cast<const uint16_t*>(p) + i);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = EK == EL_F16 ? f16_to_f32(a[e]) : bf16_to_f32(a[e]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < n ? elem_f32<EK>(p, i + e) : 0.0f;
  }
}

}  // namespace aicf::hip
