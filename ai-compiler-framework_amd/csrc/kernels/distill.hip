// Distillation from a teacher's top K logits: loss and gradient by the
// student's logits in one pass over the row.
//
//   p = softmax over the teacher's given classes of T / tau
//   row loss = (1 - a) tau^2 sum_j p_j (log p_j - log q_tau[I_j]) + a (-log q_1[label])
//     with q_tau = softmax(Z / tau), q_1 = softmax(Z)
//   loss = sum_r w_r row_loss_r
//   dZ = w [ (1 - a) tau (q_tau - p) + a (q_1 - onehot(label)) ]
//
// The gradient is dense (every class has its q) with K + 1 exceptions a row:
// the dense part is written first, the classes of the teacher and of the label
// after it, from the logits gathered before (dZ may be Z).  Sums and statistics
// are f32 (the loss over rows f64), the gradient is rounded once.
//
// No counterpart in the reference.
#include "../common/head_util.hpp"

namespace aicf::hip {

namespace {

constexpr int kMaxK = 1024;  // the teacher's classes a row (LDS)

struct DistillArgs {
  const void* z;
  const void* t;
  const int32_t* ids;
  const int32_t* labels;
  const float* w;
  void* dz;  // nullptr: the loss alone
  float* row_loss;
  int64_t R, V, ldz, ldt, ldi, lddz;
  int K;
  float tau, alpha, w0;  // w0: the weight of every row where w is absent
};

constexpr float kLog2e = 1.4426950408889634f;

// Maximum of a row segment, and the sums of exp((z - m) / tau) and exp(z - m).
struct Soft {
  float m, s, s1;
};
__device__ __forceinline__ float safe_ref(float m) { return m == -INFINITY ? 0.0f : m; }
template <bool DUAL>
__device__ __forceinline__ void soft_merge(Soft& a, const Soft& b, float c) {
  const float M = fmaxf(a.m, b.m), ref = safe_ref(M);
  a.s = a.s * __builtin_amdgcn_exp2f((a.m - ref) * c) + b.s * __builtin_amdgcn_exp2f((b.m - ref) * c);
  if constexpr (DUAL)
    a.s1 = a.s1 * __builtin_amdgcn_exp2f((a.m - ref) * kLog2e) + b.s1 * __builtin_amdgcn_exp2f((b.m - ref) * kLog2e);
  a.m = M;
}
template <bool DUAL>
__device__ __forceinline__ void soft_add8(Soft& a, const float (&v)[8], int n, float c) {
  float m = a.m;
#pragma unroll
  for (int e = 0; e < 8; ++e) m = e < n ? fmaxf(m, v[e]) : m;
  const float ref = safe_ref(m);
  float s = 0.0f, s1 = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float d = e < n ? v[e] - ref : -INFINITY;
    s += __builtin_amdgcn_exp2f(d * c);
    if constexpr (DUAL) s1 += __builtin_amdgcn_exp2f(d * kLog2e);
  }
  if (m != a.m) {
    a.s *= __builtin_amdgcn_exp2f((a.m - ref) * c);
    if constexpr (DUAL) a.s1 *= __builtin_amdgcn_exp2f((a.m - ref) * kLog2e);
    a.m = m;
  }
  a.s += s;
  if constexpr (DUAL) a.s1 += s1;
}

template <int NT>
__device__ __forceinline__ float block_max(float v, float* red) {
  v = wave_max(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int k = 1; k < NT / 64; ++k) v = fmaxf(v, red[k]);
  return v;
}
template <int NT>
__device__ __forceinline__ float block_sum(float v, float* red) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int k = 1; k < NT / 64; ++k) v += red[k];
  return v;
}

template <int EK>
__device__ __forceinline__ void put_elem(void* p, int64_t i, float v) {
  if constexpr (EK == EL_F32) static_cast<float*>(p)[i] = v;
  else static_cast<uint16_t*>(p)[i] = EK == EL_F16 ? f32_to_f16(v) : f32_to_bf16(v);
}
template <int EK>
__device__ __forceinline__ void put8(void* p, int64_t i, const float (&v)[8], int n) {
  if (n >= 8) {
    if constexpr (EK == EL_F32) {
      float* q = static_cast<float*>(p) + i;
      *reinterpret_cast<f32x4_a4*>(q) = f32x4_a4{v[0], v[1], v[2], v[3]};
      *reinterpret_cast<f32x4_a4*>(q + 4) = f32x4_a4{v[4], v[5], v[6], v[7]};
    } else {
      u16x8_a2 o;
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        if constexpr (EK == EL_BF16) {
          const uint32_t w = f32x2_to_bf16x2(v[e], v[e + 1]);
          o[e] = (uint16_t)w;
          o[e + 1] = (uint16_t)(w >> 16);
        } else {
          o[e] = f32_to_f16(v[e]);
          o[e + 1] = f32_to_f16(v[e + 1]);
        }
      }
      *reinterpret_cast<u16x8_a2*>(static_cast<uint16_t*>(p) + i) = o;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 7; ++e)
      if (e < n) put_elem<EK>(p, i + e, v[e]);
  }
}

__device__ __forceinline__ float elem_any(const void* p, int64_t i, int ek) {
  if (ek == EL_F32) return elem_f32<EL_F32>(p, i);
  return ek == EL_F16 ? elem_f32<EL_F16>(p, i) : elem_f32<EL_BF16>(p, i);
}

// One workgroup a row.
template <int NT, int EK, bool DUAL>
__global__ __launch_bounds__(NT) void distill_row_kernel(DistillArgs a, int tk) {
  __shared__ int cls[kMaxK + 1];    // the row's special classes: the teacher's, the label (-1: none)
  __shared__ float zs[kMaxK + 1];   // their logits
  __shared__ float es[kMaxK + 1];   // what the gradient has less there: (1 - a) tau p, a
  __shared__ float red[NT / 64];
  __shared__ Soft part[NT / 64];
  const int t = threadIdx.x;
  const int64_t row = blockIdx.x;
  const float w = a.w ? a.w[row] : a.w0;
  const int V = (int)a.V;
  if (w == 0.0f) {  // left out: not read
    if (a.dz) {
      const float zero[8] = {0, 0, 0, 0, 0, 0, 0, 0};
      for (int c = t * 8; c < V; c += NT * 8) put8<EK>(a.dz, row * a.lddz + c, zero, V - c);
    }
    if (t == 0) a.row_loss[row] = 0.0f;
    return;
  }
  const float c2 = kLog2e / a.tau;
  const int64_t zrow = row * a.ldz;

  // the special classes
  float tm = -INFINITY;
  for (int j = t; j < a.K; j += NT) {
    const int id = a.ids[row * a.ldi + j];
    const bool ok = id >= 0 && id < V;
    cls[j] = ok ? id : -1;
    zs[j] = ok ? elem_f32<EK>(a.z, zrow + id) : 0.0f;
    const float x = ok ? elem_any(a.t, row * a.ldt + j, tk) / a.tau : -INFINITY;
    es[j] = x;
    tm = fmaxf(tm, x);
  }
  if (t == 0) {
    const int lab = a.labels && a.alpha != 0.0f ? a.labels[row] : -1;
    const bool ok = lab >= 0 && lab < V;
    cls[a.K] = ok ? lab : -1;
    zs[a.K] = ok ? elem_f32<EK>(a.z, zrow + lab) : 0.0f;
  }
  tm = safe_ref(block_max<NT>(tm, red));

  // the row's statistics
  Soft st{-INFINITY, 0.0f, 0.0f};
  for (int c = t * 8; c < V; c += NT * 8) {
    float v[8];
    load8<EK>(v, a.z, zrow + c, V - c);
    soft_add8<DUAL>(st, v, V - c, c2);
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1)
    soft_merge<DUAL>(st, Soft{__shfl_xor(st.m, off, 64), __shfl_xor(st.s, off, 64), __shfl_xor(st.s1, off, 64)}, c2);
  if ((t & 63) == 0) part[t >> 6] = st;
  float ts = 0.0f;
  for (int j = t; j < a.K; j += NT) ts += __expf(es[j] - tm);
  ts = block_sum<NT>(ts, red);  // (its barriers order `part` too)
  st = part[0];
#pragma unroll
  for (int k = 1; k < NT / 64; ++k) soft_merge<DUAL>(st, part[k], c2);
  if (!DUAL) st.s1 = st.s;  // tau = 1, or no labels' loss
  if (st.m == -INFINITY) st.s = st.s1 = __builtin_nanf("");  // no class has any probability

  const bool some = ts > 0.0f || ts != ts;
  const bool has = cls[a.K] >= 0;
  const float soft_w = some ? (1.0f - a.alpha) * a.tau : 0.0f, hard_w = has ? a.alpha : 0.0f;
  const float lnS = logf(st.s), lnT = logf(ts), inv_t = some ? 1.0f / ts : 0.0f;
  float l = 0.0f;
  for (int j = t; j < a.K; j += NT) {
    const float x = es[j] - tm, p = cls[j] >= 0 ? __expf(x) * inv_t : 0.0f;
    if (p != 0.0f) l += p * ((x - lnT) - ((zs[j] - st.m) / a.tau - lnS));
    es[j] = soft_w * p;
  }
  if (t == 0) es[a.K] = hard_w;
  l = block_sum<NT>(l, red);
  if (t == 0) {
    float rl = (1.0f - a.alpha) * a.tau * a.tau * l;
    if (has) rl -= a.alpha * ((zs[a.K] - st.m) - logf(st.s1));
    a.row_loss[row] = rl;
  }
  if (!a.dz) return;

  // the dense part
  const float k1 = w * hard_w / st.s1, k2 = w * soft_w / st.s + (DUAL ? 0.0f : k1);
  auto dense = [&](float z) {
    const float d = z - st.m;
    float g = k2 * __builtin_amdgcn_exp2f(d * c2);
    if constexpr (DUAL) g = fmaf(k1, __builtin_amdgcn_exp2f(d * kLog2e), g);
    return g;
  };
  for (int c = t * 8; c < V; c += NT * 8) {
    float v[8];
    load8<EK>(v, a.z, zrow + c, V - c);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = dense(v[e]);
    put8<EK>(a.dz, row * a.lddz + c, v, V - c);
  }
  __syncthreads();  // the special classes' dense values are stored
  for (int j = t; j <= a.K; j += NT) {
    const int id = cls[j];
    float e = 0.0f;
    bool first = id >= 0;
    for (int i = 0; i <= a.K; ++i) {
      if (cls[i] == id) {
        e += es[i];
        first = first && i >= j;
      }
    }
    if (first) put_elem<EK>(a.dz, row * a.lddz + id, dense(zs[j]) - w * e);
  }
}

// loss = sum of w_r row_loss_r, f64 in a fixed order (one workgroup).
__global__ __launch_bounds__(256) void distill_loss_kernel(const float* __restrict__ rl, const float* __restrict__ w,
                                                           float w0, int64_t R, float* __restrict__ loss) {
  __shared__ double red[4];
  double s = 0.0;
  for (int64_t r = threadIdx.x; r < R; r += 256) s += (double)(w ? w[r] : w0) * (double)rl[r];
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) loss[0] = (float)((red[0] + red[1]) + (red[2] + red[3]));
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
struct DistillCall {
  const TensorDesc *z, *t, *ids, *labels, *w;
  const TensorDesc *loss, *dz, *row_loss, *scratch;
  float tau, alpha;
};

bool distill_read(const TensorDesc* in, int ni, const TensorDesc* out, int no, const void* attr, DistillCall& c) {
  if (!in || !out || ni < 3 || ni > 5 || no < 2 || no > 4) return false;
  const AttrBlob& b = blob(attr);
  c = DistillCall{};
  c.tau = 1.0f;
  if (b.schema_id == AICF_SCHEMA_DTOP) {
    if (!payload_ok(b, 8)) return false;
    c.tau = field<float>(b, 0);
    c.alpha = field<float>(b, 4);
  }
  if (!(c.tau > 0.0f && c.tau <= 3.0e38f) || !(c.alpha >= 0.0f && c.alpha <= 1.0f)) return false;
  c.z = in;
  c.t = in + 1;
  c.ids = in + 2;
  for (int i = 3; i < ni; ++i) {
    if (dt(in[i]) == DType::kI32 && i == 3) c.labels = in + i;
    else if (dt(in[i]) == DType::kF32 && i == ni - 1) c.w = in + i;
    else return false;
  }
  c.loss = out;
  int k = 1;
  if (out[k].rank == 2) c.dz = out + k++;
  if (k >= no) return false;
  c.row_loss = out + k++;
  if (k < no) c.scratch = out + k++;
  return k == no;
}

bool distill_sup(const TensorDesc* in, int ni, const TensorDesc* out, int no, const void* attr) {
  DistillCall c;
  if (!distill_read(in, ni, out, no, attr, c)) return false;
  int ek, tk;
  int64_t ld;
  if (!elem_kind(*c.z, &ek) || !matrix_ld(*c.z, false, &ld)) return false;
  const int64_t R = c.z->shape[0], V = c.z->shape[1];
  if (R < 1 || V < 1 || R > INT32_MAX || V > INT32_MAX - (1 << 16)) return false;
  if (!elem_kind(*c.t, &tk) || !matrix_ld(*c.t, false, &ld)) return false;
  const int64_t K = c.t->shape[1];
  if (c.t->shape[0] != R || K < 1 || K > kMaxK) return false;
  if (dt(*c.ids) != DType::kI32 || !matrix_ld(*c.ids, false, &ld) || !same_shape(*c.ids, *c.t)) return false;
  if (c.labels && !vector_of(*c.labels, DType::kI32, R)) return false;
  if (c.w && !vector_of(*c.w, DType::kF32, R)) return false;
  if (dt(*c.loss) != DType::kF32 || numel_of(*c.loss) != 1) return false;
  if (c.dz && (c.dz->dtype != c.z->dtype || !matrix_ld(*c.dz, true, &ld) || !same_shape(*c.dz, *c.z))) return false;
  if (!vector_of(*c.row_loss, DType::kF32, R)) return false;
  if (c.scratch) {
    const TensorDesc& s = *c.scratch;
    if (dt(s) != DType::kF32 || s.rank != 3 || !s.contiguous || s.shape[0] != R || s.shape[1] < 2 || s.shape[2] != 4)
      return false;
  }
  // outputs apart from the inputs and from one another; dZ may be Z itself
  for (int i = 0; i < no; ++i) {
    for (int j = 0; j < ni; ++j) {
      if (out + i == c.dz && j == 0 && out[i].data == in[j].data && R * V > 0) {
        int64_t lz, ldz;
        matrix_ld(*c.z, false, &lz);
        matrix_ld(*c.dz, true, &ldz);
        if (lz == ldz) continue;
      }
      if (views_overlap(out[i], in[j])) return false;
    }
    for (int j = 0; j < i; ++j)
      if (views_overlap(out[i], out[j])) return false;
  }
  return true;
}

template <int EK, bool DUAL>
Status distill_rows(const DistillArgs& a, int tk, hipStream_t s) {
  // a grid's lanes are counted in 32 bits
  const int nt = a.V > 8192 ? 1024 : 256;
  const int64_t step = (int64_t{1} << 31) / nt;
  for (int64_t r = 0; r < a.R; r += step) {
    DistillArgs p = a;
    p.R = a.R - r < step ? a.R - r : step;
    const int64_t es = EK == EL_F32 ? 4 : 2, et = tk == EL_F32 ? 4 : 2;
    p.z = (const uint8_t*)a.z + r * a.ldz * es;
    p.t = (const uint8_t*)a.t + r * a.ldt * et;
    p.ids = a.ids + r * a.ldi;
    if (a.labels) p.labels = a.labels + r;
    if (a.w) p.w = a.w + r;
    if (a.dz) p.dz = (uint8_t*)a.dz + r * a.lddz * es;
    p.row_loss = a.row_loss + r;
    if (nt == 1024) distill_row_kernel<1024, EK, DUAL><<<(unsigned)p.R, 1024, 0, s>>>(p, tk);
    else distill_row_kernel<256, EK, DUAL><<<(unsigned)p.R, 256, 0, s>>>(p, tk);
    const Status st = launch_status("distill_topk");
    if (st != Status::Ok) return st;
  }
  return Status::Ok;
}

Status distill_launch(const TensorDesc* in, int ni, TensorDesc* out, int no, const void* at, void*, size_t,
                      void* stream) {
  if (!distill_sup(in, ni, out, no, at)) return Status::InvalidArgument;
  for (int k = 0; k < ni; ++k)
    if (no_memory(in[k])) return Status::InvalidArgument;
  for (int k = 0; k < no; ++k)
    if (no_memory(out[k])) return Status::InvalidArgument;
  DistillCall c;
  distill_read(in, ni, out, no, at, c);
  DistillArgs a{};
  a.R = c.z->shape[0];
  a.V = c.z->shape[1];
  a.K = (int)c.t->shape[1];
  a.z = c.z->data;
  a.t = c.t->data;
  a.ids = (const int32_t*)c.ids->data;
  a.labels = c.labels ? (const int32_t*)c.labels->data : nullptr;
  a.w = c.w ? (const float*)c.w->data : nullptr;
  a.w0 = 1.0f / (float)a.R;
  a.dz = c.dz ? c.dz->data : nullptr;
  a.row_loss = (float*)c.row_loss->data;
  matrix_ld(*c.z, false, &a.ldz);
  matrix_ld(*c.t, false, &a.ldt);
  matrix_ld(*c.ids, false, &a.ldi);
  if (c.dz) matrix_ld(*c.dz, true, &a.lddz);
  a.tau = c.tau;
  a.alpha = c.alpha;
  int ek, tk;
  elem_kind(*c.z, &ek);
  elem_kind(*c.t, &tk);
  hipStream_t s = as_stream(stream);
  const bool dual = a.labels && a.alpha != 0.0f && a.tau != 1.0f;
  Status st;
  if (ek == EL_F32) st = dual ? distill_rows<EL_F32, true>(a, tk, s) : distill_rows<EL_F32, false>(a, tk, s);
  else if (ek == EL_F16) st = dual ? distill_rows<EL_F16, true>(a, tk, s) : distill_rows<EL_F16, false>(a, tk, s);
  else st = dual ? distill_rows<EL_BF16, true>(a, tk, s) : distill_rows<EL_BF16, false>(a, tk, s);
  if (st != Status::Ok) return st;
  distill_loss_kernel<<<1, 256, 0, s>>>(a.row_loss, a.w, a.w0, a.R, (float*)c.loss->data);
  return launch_status("distill_loss");
}

size_t no_workspace(const TensorDesc*, int, const void*) { return 0; }

}  // namespace

KernelVariant make_distill_topk_variant() {
  KernelVariant v;
  v.name = "distill_topk";
  v.launch = distill_launch;
  v.supported = distill_sup;
  v.query_workspace = no_workspace;
  return v;
}

}  // namespace aicf::hip
