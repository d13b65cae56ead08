// The norm of a model's gradients over all tensors, the factor that clips it,
// and the clipped gradients.
//
//   norm = sqrt(sum over tensors and elements of g^2)
//   factor = min(1, max_norm / (norm + 1e-6))
//   G' = factor G (in place or elsewhere), rounded once
//
// One pass reads every gradient once (bound by memory: 2 operations an
// element), a second workgroup-sized launch joins the partial sums, and the
// clipping reads and writes once more (the other way round, so that it begins
// with what the last-level cache still holds); in place with factor 1 it touches
// nothing.  A launch takes a table of tensors by value, so nothing is copied to
// the device and the call can be captured.  Squares and sums are f64: exact squares
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

constexpr int kScratchTensors = 96;  // partial sums of a call: kBlocks for each 96 tensors
constexpr int kBlocks = 1024;        // workgroups a launch at most
// Tensors a launch: 3.6 and 3.9 KB of kernel arguments.
constexpr int kNormTable = 256, kClipTable = 176;

// A workgroup's step, an item, is kRow H 16-bit elements of a tensor (f32: half
// as many, but kRow at least), 8 a lane and load, all loaded at once.  H = 4, or
// 1 where that left workgroups without an item.
constexpr int kThreads = 512, kRow = 8 * kThreads;
__host__ __device__ __forceinline__ int item_of(int kind, int H) { return kRow * (kind == EL_F32 ? (H + 1) / 2 : H); }

template <int N, bool OUT>
struct NormTable {
  const void* g[N];
  void* out[OUT ? N : 1];
  int32_t start[N + 1];  // items before a tensor
  uint16_t last[N];      // elements of its last item - 1, and its type << 14
  int count;

  __device__ __forceinline__ int kind(int k) const { return last[k] >> 14; }
  __device__ __forceinline__ int64_t numel(int k, int per) const {
    return (int64_t)(start[k + 1] - start[k] - 1) * per + (last[k] & 0x3fff) + 1;
  }
  // The tensor that item i belongs to.
  __device__ __forceinline__ int tensor_of(int i) const {
    int lo = 0, hi = count - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (start[mid] <= i) lo = mid;
      else hi = mid - 1;
    }
    return lo;
  }
};

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

template <int EK, int H>
__device__ __forceinline__ void squares(const void* g, int64_t at, int64_t n, double (&acc)[2]) {
  float v[H][8];
#pragma unroll
  for (int h = 0; h < H; ++h) load8<EK>(v[h], g, at + h * kRow + threadIdx.x * 8, n - h * kRow - threadIdx.x * 8);
#pragma unroll
  for (int h = 0; h < H; ++h)
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[h & 1] = fma((double)v[h][e], (double)v[h][e], acc[h & 1]);
}

// Workgroup b takes items b per .. (b + 1) per - 1.
template <int H>
__global__ __launch_bounds__(kThreads) void norm_part_kernel(NormTable<kNormTable, false> t, int per,
                                                             double* __restrict__ partial) {
  __shared__ double red[kThreads / 64];
  const int first = blockIdx.x * per, last = first + per < t.start[t.count] ? first + per : t.start[t.count];
  double acc[2] = {0.0, 0.0};
  int k = first < last ? t.tensor_of(first) : 0;
  for (int i = first; i < last; ++i) {
    while (i >= t.start[k + 1]) ++k;
    const int item = item_of(t.kind(k), H);
    const int64_t at = (int64_t)(i - t.start[k]) * item, n = t.numel(k, item) - at;
    if (t.kind(k) == EL_F32) squares<EL_F32, (H + 1) / 2>(t.g[k], at, n, acc);
    else if (t.kind(k) == EL_F16) squares<EL_F16, H>(t.g[k], at, n, acc);
    else squares<EL_BF16, H>(t.g[k], at, n, acc);
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

template <int EK, int H>
__device__ __forceinline__ void scaled(const void* g, void* out, int64_t at, int64_t n, float f) {
  float v[H][8];
#pragma unroll
  for (int h = 0; h < H; ++h) load8<EK>(v[h], g, at + h * kRow + threadIdx.x * 8, n - h * kRow - threadIdx.x * 8);
#pragma unroll
  for (int h = 0; h < H; ++h) {
    const int64_t i = at + h * kRow + threadIdx.x * 8, left = n - h * kRow - threadIdx.x * 8;
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

template <int H>
__global__ __launch_bounds__(kThreads) void norm_clip_kernel(NormTable<kClipTable, true> t, int per,
                                                             const float* __restrict__ norm) {
  const float f = norm[1];
  const int first = (gridDim.x - 1 - blockIdx.x) * per;
  const int last = first + per < t.start[t.count] ? first + per : t.start[t.count];
  int k = first < last ? t.tensor_of(first) : 0;
  for (int i = first; i < last; ++i) {
    while (i >= t.start[k + 1]) ++k;
    if (f == 1.0f && t.g[k] == t.out[k]) continue;
    const int item = item_of(t.kind(k), H);
    const int64_t at = (int64_t)(i - t.start[k]) * item, n = t.numel(k, item) - at;
    if (t.kind(k) == EL_F32) scaled<EL_F32, (H + 1) / 2>(t.g[k], t.out[k], at, n, f);
    else if (t.kind(k) == EL_F16) scaled<EL_F16, H>(t.g[k], t.out[k], at, n, f);
    else scaled<EL_BF16, H>(t.g[k], t.out[k], at, n, f);
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

int64_t norm_scratch(int T) { return (int64_t)2 * kBlocks * ((T + kScratchTensors - 1) / kScratchTensors); }

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
  int64_t bytes = 0;
  for (int k = 0; k < ni; ++k) bytes += numel_of(in[k]) * (dt(in[k]) == DType::kF32 ? 4 : 2);
  const int h = bytes >= (int64_t)8 * kRow * kBlocks ? 4 : 1;
  // tensors k0 .. in a table: f(table, items of a workgroup, workgroups)
  auto table = [&](auto t, int N, int k0, auto f) {
    t.count = 0;
    t.start[0] = 0;
    for (int k = k0; k < ni && k < k0 + N; ++k) {
      const int64_t n = numel_of(in[k]);
      if (n == 0) continue;
      int ek;
      elem_kind(in[k], &ek);
      const int64_t item = item_of(ek, h);
      t.g[t.count] = in[k].data;
      if (N == kClipTable) t.out[t.count] = out[2 + k].data;
      t.last[t.count] = (uint16_t)((n - 1) % item | ek << 14);
      t.start[t.count + 1] = t.start[t.count] + (int32_t)((n + item - 1) / item);
      ++t.count;
    }
    const int items = t.start[t.count], per = (items + kBlocks - 1) / kBlocks;
    if (items > 0) f(t, per, (unsigned)((items + per - 1) / per));
  };
  int parts = 0;
  for (int k0 = 0; k0 < ni; k0 += kNormTable)
    table(NormTable<kNormTable, false>(), kNormTable, k0, [&](const auto& t, int per, unsigned blocks) {
      if (h == 4) norm_part_kernel<4><<<blocks, kThreads, 0, s>>>(t, per, partial + parts);
      else norm_part_kernel<1><<<blocks, kThreads, 0, s>>>(t, per, partial + parts);
      parts += (int)blocks;
    });
  norm_join_kernel<<<1, 1024, 0, s>>>(partial, parts, max_norm, norm);
  if (no > 2)
    for (int k0 = (ni - 1) / kClipTable * kClipTable; k0 >= 0; k0 -= kClipTable)
      table(NormTable<kClipTable, true>(), kClipTable, k0, [&](const auto& t, int per, unsigned blocks) {
        if (h == 4) norm_clip_kernel<4><<<blocks, kThreads, 0, s>>>(t, per, norm);
        else norm_clip_kernel<1><<<blocks, kThreads, 0, s>>>(t, per, norm);
      });
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
