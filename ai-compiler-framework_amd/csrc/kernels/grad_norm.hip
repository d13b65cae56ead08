// The norm of a model's gradients over all tensors, the factor that clips it,
// and the clipped gradients.
//
//   norm = sqrt(sum over tensors and elements of g^2)
//   factor = min(1, max_norm / (norm + 1e-6))
//   G' = factor G (in place or elsewhere), rounded once
//
// One pass reads every gradient once (bound by memory: 2 operations an
// element), a second workgroup-sized launch joins the partial sums, and the
// clipping reads and writes once more; in place with factor 1 it touches
// nothing.  A launch takes kTable tensors by value, so nothing is copied to the
// device and the call can be captured.  Squares and sums are f64: exact squares
// of any f32, no overflow or underflow where the norm itself has none, and the
// same bits whatever scale the gradients are at; the loads bound the pass all
// the same.  Every sum has a fixed order.
//
// No counterpart in the reference.
#include <algorithm>
#include <exception>
#include <vector>

#include "../common/head_util.hpp"

namespace aicf::hip {

namespace {

constexpr int kTable = 96;      // tensors a launch (2.8 KB of kernel arguments)
constexpr int kItem = 4096;     // elements of a workgroup's step: 16 a lane
constexpr int kBlocks = 1024;   // workgroups a launch at most: partial sums of a call are kBlocks a launch

struct NormTable {
  const void* g[kTable];
  void* out[kTable];
  int64_t n[kTable];
  int32_t start[kTable + 1];  // items before a tensor
  uint8_t kind[kTable];
  int count;
};

// The tensor that item belongs to.
__device__ __forceinline__ int tensor_of(const NormTable& t, int item) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.start[mid] <= item) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ double block_sum_f64(double v, double* red) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  const int w = threadIdx.x >> 6, nw = blockDim.x >> 6;
  if ((threadIdx.x & 63) == 0) red[w] = v;
  __syncthreads();
  v = red[0];
  for (int i = 1; i < nw; ++i) v += red[i];
  return v;
}

template <int EK>
__device__ __forceinline__ void squares(const void* g, int64_t at, int64_t n, double (&acc)[2]) {
  float v[2][8];
  load8<EK>(v[0], g, at + threadIdx.x * 8, n - threadIdx.x * 8);
  load8<EK>(v[1], g, at + 2048 + threadIdx.x * 8, n - 2048 - threadIdx.x * 8);
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[h] = fma((double)v[h][e], (double)v[h][e], acc[h]);
}

// Workgroup b takes items b per .. (b + 1) per - 1.
__global__ __launch_bounds__(256) void norm_part_kernel(NormTable t, int per, double* __restrict__ partial) {
  __shared__ double red[4];
  const int first = blockIdx.x * per, last = first + per < t.start[t.count] ? first + per : t.start[t.count];
  double acc[2] = {0.0, 0.0};
  int k = first < last ? tensor_of(t, first) : 0;
  for (int i = first; i < last; ++i) {
    while (i >= t.start[k + 1]) ++k;
    const int64_t at = (int64_t)(i - t.start[k]) * kItem, n = t.n[k] - at;
    if (t.kind[k] == EL_F32) squares<EL_F32>(t.g[k], at, n, acc);
    else if (t.kind[k] == EL_F16) squares<EL_F16>(t.g[k], at, n, acc);
    else squares<EL_BF16>(t.g[k], at, n, acc);
  }
  const double v = block_sum_f64(acc[0] + acc[1], red);
  if (threadIdx.x == 0) partial[blockIdx.x] = v;
}

__global__ __launch_bounds__(1024) void norm_join_kernel(const double* __restrict__ partial, int parts, float max_norm,
                                                         float* __restrict__ norm) {
  __shared__ double red[16];
  double v = 0.0;
  for (int i = threadIdx.x; i < parts; i += 1024) v += partial[i];
  v = block_sum_f64(v, red);
  if (threadIdx.x == 0) {
    const double l = sqrt(v), f = (double)max_norm / (l + 1e-6);
    norm[0] = (float)l;
    norm[1] = f < 1.0 || f != f ? (float)f : 1.0f;
  }
}

template <int EK>
__device__ __forceinline__ void scaled(const void* g, void* out, int64_t at, int64_t n, float f) {
  float v[2][8];
  load8<EK>(v[0], g, at + threadIdx.x * 8, n - threadIdx.x * 8);
  load8<EK>(v[1], g, at + 2048 + threadIdx.x * 8, n - 2048 - threadIdx.x * 8);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int64_t i = at + h * 2048 + threadIdx.x * 8, left = n - h * 2048 - threadIdx.x * 8;
    if constexpr (EK == EL_F32) {
      float* q = (float*)out + i;
      if (left >= 8) {
        *reinterpret_cast<f32x4_a4*>(q) = f32x4_a4{v[h][0] * f, v[h][1] * f, v[h][2] * f, v[h][3] * f};
        *reinterpret_cast<f32x4_a4*>(q + 4) = f32x4_a4{v[h][4] * f, v[h][5] * f, v[h][6] * f, v[h][7] * f};
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e < left) q[e] = v[h][e] * f;
      }
    } else {
      uint16_t* q = (uint16_t*)out + i;
      u16x8_a2 o;
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = EK == EL_F16 ? f32_to_f16(v[h][e] * f) : f32_to_bf16(v[h][e] * f);
      if (left >= 8) {
        *reinterpret_cast<u16x8_a2*>(q) = o;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e < left) q[e] = o[e];
      }
    }
  }
}

__global__ __launch_bounds__(256) void norm_clip_kernel(NormTable t, int per, const float* __restrict__ norm) {
  const float f = norm[1];
  const int first = blockIdx.x * per, last = first + per < t.start[t.count] ? first + per : t.start[t.count];
  int k = first < last ? tensor_of(t, first) : 0;
  for (int i = first; i < last; ++i) {
    while (i >= t.start[k + 1]) ++k;
    if (f == 1.0f && t.g[k] == t.out[k]) continue;
    const int64_t at = (int64_t)(i - t.start[k]) * kItem, n = t.n[k] - at;
    if (t.kind[k] == EL_F32) scaled<EL_F32>(t.g[k], t.out[k], at, n, f);
    else if (t.kind[k] == EL_F16) scaled<EL_F16>(t.g[k], t.out[k], at, n, f);
    else scaled<EL_BF16>(t.g[k], t.out[k], at, n, f);
  }
}

// ---------------------------------------------------------------------------
// Host side: G_1 .. G_T -> norm [2], scratch [, G'_1 .. G'_T]
// ---------------------------------------------------------------------------
bool norm_attr(const void* attr, float* max_norm) {
  const AttrBlob& a = blob(attr);
  if (!attr || a.schema_id != AICF_SCHEMA_GNRM || a.bytes != 4 || !a.data) return false;
  *max_norm = field<float>(a, 0);
  return *max_norm >= 0.0f;  // (no NaN)
}

bool row_major(const TensorDesc& t) {
  if (t.rank < 0 || t.rank > AICF_MAX_RANK) return false;
  int64_t n = 1;
  for (int i = t.rank - 1; i >= 0; --i) {
    if (t.shape[i] < 0 || (t.shape[i] > 1 && n > 0 && t.stride[i] != n)) return false;
    if (__builtin_mul_overflow(n, t.shape[i], &n) || n > (int64_t)1 << 42) return false;
  }
  return true;
}

int64_t norm_scratch(int T) { return (int64_t)2 * kBlocks * ((T + kTable - 1) / kTable); }

bool norm_sup(const TensorDesc* in, int ni, const TensorDesc* out, int no, const void* attr) {
  float max_norm;
  if (!in || !out || ni < 1 || ni > 65536 || (no != 2 && no != 2 + ni) || !norm_attr(attr, &max_norm)) return false;
  if (!vector_of(out[0], DType::kF32, 2)) return false;
  const TensorDesc& sc = out[1];
  if (dt(sc) != DType::kF32 || sc.rank != 1 || sc.shape[0] < norm_scratch(ni) || sc.stride[0] != 1) return false;
  if (!aligned(sc.data, 8)) return false;
  // spans of what is written (bit 0) and read (bit 1), by address: a written one meets no other, but G' its own G
  struct Part {
    Span s;
    bool written;
  };
  std::vector<Part> parts;
  try {
    parts.reserve(2 * (size_t)ni + 2);
  } catch (const std::exception&) {
    return false;
  }
  int64_t total = 0;
  for (int k = 0; k < ni; ++k) {
    int ek;
    if (!elem_kind(in[k], &ek) || !row_major(in[k])) return false;
    total += numel_of(in[k]);
    if (total > (int64_t)1 << 42) return false;  // items are counted in 32 bits
    const bool same = no > 2 && out[2 + k].data == in[k].data;
    if (no > 2) {
      const TensorDesc& o = out[2 + k];
      if (dt(o) != dt(in[k]) || !row_major(o) || !same_shape(o, in[k])) return false;
      if (numel_of(o) > 0) parts.push_back({span_of(o), true});
    }
    if (!same && numel_of(in[k]) > 0) parts.push_back({span_of(in[k]), false});
  }
  parts.push_back({span_of(out[0]), true});
  parts.push_back({span_of(sc), true});
  std::sort(parts.begin(), parts.end(), [](const Part& a, const Part& b) { return a.s.lo < b.s.lo; });
  uintptr_t end = 0, end_written = 0;  // of all before, of the written ones before
  for (const Part& q : parts) {
    if (q.s.lo < end_written || (q.written && q.s.lo < end)) return false;
    end = std::max(end, q.s.hi);
    if (q.written) end_written = std::max(end_written, q.s.hi);
  }
  return true;
}

Status norm_launch(const TensorDesc* in, int ni, TensorDesc* out, int no, const void* attr, void*, size_t,
                   void* stream) {
  if (!norm_sup(in, ni, out, no, attr)) return Status::InvalidArgument;
  for (int k = 0; k < ni; ++k)
    if (no_memory(in[k])) return Status::InvalidArgument;
  for (int k = 0; k < no; ++k)
    if (no_memory(out[k])) return Status::InvalidArgument;
  float max_norm = 0.0f;
  norm_attr(attr, &max_norm);
  hipStream_t s = as_stream(stream);
  float* norm = (float*)out[0].data;
  double* partial = (double*)out[1].data;
  // launches of kTable tensors each: f(table, items of a workgroup, workgroups)
  auto tables = [&](auto f) {
    NormTable t;
    for (int k0 = 0; k0 < ni; k0 += kTable) {
      t.count = 0;
      t.start[0] = 0;
      for (int k = k0; k < ni && k < k0 + kTable; ++k) {
        const int64_t n = numel_of(in[k]);
        if (n == 0) continue;
        int ek;
        elem_kind(in[k], &ek);
        t.g[t.count] = in[k].data;
        t.out[t.count] = no > 2 ? out[2 + k].data : nullptr;
        t.n[t.count] = n;
        t.kind[t.count] = (uint8_t)ek;
        t.start[t.count + 1] = t.start[t.count] + (int32_t)((n + kItem - 1) / kItem);
        ++t.count;
      }
      const int items = t.start[t.count], per = (items + kBlocks - 1) / kBlocks;
      if (items > 0) f(t, per, (unsigned)((items + per - 1) / per));
    }
  };
  int parts = 0;
  tables([&](const NormTable& t, int per, unsigned blocks) {
    norm_part_kernel<<<blocks, 256, 0, s>>>(t, per, partial + parts);
    parts += (int)blocks;
  });
  norm_join_kernel<<<1, 1024, 0, s>>>(partial, parts, max_norm, norm);
  if (no > 2)
    tables([&](const NormTable& t, int per, unsigned blocks) { norm_clip_kernel<<<blocks, 256, 0, s>>>(t, per, norm); });
  return launch_status("grad_norm");
}

size_t no_workspace(const TensorDesc*, int, const void*) { return 0; }

}  // namespace

KernelVariant make_grad_norm_variant() {
  KernelVariant v;
  v.name = "grad_norm";
  v.expected_attr_schema_id = AICF_SCHEMA_GNRM;
  v.launch = norm_launch;
  v.supported = norm_sup;
  v.query_workspace = no_workspace;
  return v;
}

}  // namespace aicf::hip
