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

#include <type_traits>

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
  float c2;              // log2(e) / tau, rounded once
};

typedef int i32x4_d __attribute__((ext_vector_type(4)));
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float safe_ref(float m) { return m == -INFINITY ? 0.0f : m; }
// 2^((z - m) c).  The difference comes first, so that the exponent is off by
// roundings of itself alone: z c - m c in one multiply-add is off by a rounding of
// m c, which differs from part to part of a row (1e-4 near logits of 1000), and is
// not a number where m c passes the type's range (rows masked with the lowest value).
// The teacher's the same.  (One more operation a class and pass: 4096 x 32000 bf16
// 105.8 -> 106.7 us, 1023 x 50021 f32 with labels 98.8 -> 100.3.)
__device__ __forceinline__ float exp_of(float z, float c, float m) { return __builtin_amdgcn_exp2f((z - m) * c); }

// Up to three values over the workgroup at once, in a fixed order (lds: 4
// floats a wave).  OP 0: maxima, 1: sums.
template <int OP, int N>
__device__ __forceinline__ void block_reduce(float (&v)[N], float* lds) {
  const int nw = blockDim.x >> 6;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = OP == 0 ? wave_max(v[i]) : wave_sum(v[i]);
  if (nw == 1) {
    __syncthreads();  // (what the callers left in LDS)
    return;
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) lds[(threadIdx.x >> 6) * 4 + i] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = lds[i];
  for (int k = 1; k < nw; ++k)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = OP == 0 ? fmaxf(v[i], lds[k * 4 + i]) : v[i] + lds[k * 4 + i];
}

// Columns of a 16-byte vector.
constexpr int width(int ek) { return ek == EL_F32 ? 4 : 8; }

template <int EK>
__device__ __forceinline__ void put_elem(void* p, int64_t i, float v) {
  if constexpr (EK == EL_F32) static_cast<float*>(p)[i] = v;
  else static_cast<uint16_t*>(p)[i] = EK == EL_F16 ? f32_to_f16(v) : f32_to_bf16(v);
}
// STREAM: loads and stores of a row with the nontemporal hint, where it is held in
// registers and nothing is read again (without it: 4096 x 32000 bf16 118.4 us,
// with it 106.9; rows at odd addresses 128.8, 123.3; f32 1023 x 50021 99.4, 96.0,
// 4096 x 50021 at odd addresses 334.6, 345.2, on 128-byte lines 326.9, 318.3).  A
// wave's accesses have to cover their lines whole: with two 16-byte vectors a lane
// in a row f32 took 461.
// (Not templates of the vector's type: that would lose its alignment.)
template <bool STREAM>
__device__ __forceinline__ f32x4 vec_load(const f32x4_a4* p) {
  if constexpr (STREAM) return __builtin_nontemporal_load(p);
  else return *p;
}
template <bool STREAM>
__device__ __forceinline__ u16x8_a2 vec_load(const u16x8_a2* p) {
  if constexpr (STREAM) return __builtin_nontemporal_load(p);
  else return *p;
}
template <bool STREAM>
__device__ __forceinline__ void vec_store(f32x4_a4* p, f32x4 v) {
  if constexpr (STREAM) __builtin_nontemporal_store(v, p);
  else *p = v;
}
template <bool STREAM>
__device__ __forceinline__ void vec_store(u16x8_a2* p, u16x8_a2 v) {
  if constexpr (STREAM) __builtin_nontemporal_store(v, p);
  else *p = v;
}
template <int EK, bool STREAM = false>
__device__ __forceinline__ void put_vec(void* p, int64_t i, const float (&v)[width(EK)], int n) {
  constexpr int W = width(EK);
  if (n >= W) {
    if constexpr (EK == EL_F32) {
      vec_store<STREAM>(reinterpret_cast<f32x4_a4*>(static_cast<float*>(p) + i), f32x4_a4{v[0], v[1], v[2], v[3]});
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
      vec_store<STREAM>(reinterpret_cast<u16x8_a2*>(static_cast<uint16_t*>(p) + i), o);
    }
  } else {
#pragma unroll
    for (int e = 0; e < W - 1; ++e)
      if (e < n) put_elem<EK>(p, i + e, v[e]);
  }
}

__device__ __forceinline__ float elem_any(const void* p, int64_t i, int ek) {
  if (ek == EL_F32) return elem_f32<EL_F32>(p, i);
  return ek == EL_F16 ? elem_f32<EL_F16>(p, i) : elem_f32<EL_BF16>(p, i);
}

// 16 bytes of logits as they are stored.
template <int EK>
struct Vec {
  typedef uint16_t u16x8v __attribute__((ext_vector_type(8)));
  static constexpr uint16_t NONE = EK == EL_F16 ? 0xfc00 : 0xff80;  // -inf
  u16x8v h;
  // elements i .. i + 7 of the columns at p
  template <bool STREAM>
  __device__ __forceinline__ void load(const uint8_t* p, int i) {
    h = vec_load<STREAM>(reinterpret_cast<const u16x8_a2*>(p + (uint32_t)i * 2u));
  }
  __device__ __forceinline__ void load_first(const uint8_t* p, int n) {  // n < 8 of them
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = e < n ? reinterpret_cast<const uint16_t*>(p)[e] : NONE;
  }
  __device__ __forceinline__ void drop(int n) {  // the first n become -inf
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = e < n ? NONE : h[e];
  }
  // What a pass made of the values is not kept for the next one.
  __device__ __forceinline__ void forget() { asm volatile("" : "+v"(h)); }
  __device__ __forceinline__ float operator[](int e) const { return EK == EL_F16 ? f16_to_f32(h[e]) : bf16_to_f32(h[e]); }
};
template <>
struct Vec<EL_F32> {
  f32x4 a;
  template <bool STREAM>
  __device__ __forceinline__ void load(const uint8_t* p, int i) {
    a = vec_load<STREAM>(reinterpret_cast<const f32x4_a4*>(p + (uint32_t)i * 4u));
  }
  __device__ __forceinline__ void load_first(const uint8_t* p, int n) {
#pragma unroll
    for (int e = 0; e < 4; ++e) a[e] = e < n ? reinterpret_cast<const float*>(p)[e] : -INFINITY;
  }
  __device__ __forceinline__ void drop(int n) {
#pragma unroll
    for (int e = 0; e < 4; ++e) a[e] = e < n ? -INFINITY : a[e];
  }
  __device__ __forceinline__ void forget() { asm volatile("" : "+v"(a)); }
  __device__ __forceinline__ float operator[](int e) const { return a[e]; }
};

// A workgroup's columns of a row, n of them: in registers (VPT vectors a
// thread; with WHOLE the first half of them, rounded down to 8 columns, lies inside), or (VPT 0) read again
// in each pass.  A vector that would pass the end is moved back to end there;
// its elements that an earlier vector holds become -inf, which adds nothing to a
// maximum or a sum, and are not stored.
template <int NT, int EK, int VPT, bool WHOLE, bool STREAM_>
struct Part {
  static constexpr bool STREAM = STREAM_;
  static constexpr int W = width(EK), INNER = WHOLE ? VPT * W / 8 / 2 * (8 / W) : 0;
  const uint8_t* z;  // the first column
  int n;
  Vec<EK> v[VPT > 0 ? VPT : 1];
  __device__ __forceinline__ int first(int k) const { return (k * NT + (int)threadIdx.x) * W; }
  __device__ __forceinline__ static bool inner(int k) { return k < INNER; }
  __device__ __forceinline__ bool beyond(int k) const { return !inner(k) && k > 0 && k * NT * W >= n; }  // uniform
  __device__ __forceinline__ int col(int k) const { return inner(k) ? first(k) : n >= W ? min(first(k), n - W) : 0; }
  // the elements [lo, hi) of vector k are its own
  __device__ __forceinline__ int lo(int k) const { return inner(k) ? 0 : min(first(k) - col(k), W); }
  __device__ __forceinline__ int hi() const { return n >= W ? W : (n > 0 ? n : 0); }
  __device__ __forceinline__ void fetch(Vec<EK>& x, int k) const {
    if (inner(k) || n >= W) {
      x.template load<STREAM>(z, col(k));
      if (!inner(k) && (k + 1) * NT * W > n) x.drop(lo(k));  // (uniform)
    } else {
      x.load_first(z, first(k) == 0 ? n : 0);
    }
  }
  __device__ __forceinline__ void open(const void* base, int64_t row, int c0, int c1) {
    z = static_cast<const uint8_t*>(base) + (row + c0) * (EK == EL_F32 ? 4 : 2);
    n = c1 - c0;
    if constexpr (VPT > 0) {
#pragma unroll
      for (int k = 0; k < VPT; ++k)
        if (!beyond(k)) fetch(v[k], k);
    }
  }
  // f(vector, its column, lo)
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    if constexpr (VPT > 0) {
#pragma unroll
      for (int k = 0; k < VPT; ++k) {
        if (!beyond(k)) f(v[k], col(k), lo(k));
        __builtin_amdgcn_sched_barrier(0);  // a vector at a time: the row's registers leave little else
      }
    } else {
      for (int k = 0; first(k) < n; k += 2) {  // two vectors on their way
        Vec<EK> x, y;
        const bool two = first(k + 1) < n;
        fetch(x, k);
        if (two) fetch(y, k + 1);
        f(x, col(k), lo(k));
        if (two) f(y, col(k + 1), lo(k + 1));
      }
    }
  }
  // Between two passes over registers: the compiler would keep the first one's
  // conversions and exponentials, several registers for each that holds the row.
  __device__ __forceinline__ void forget() {
    if constexpr (VPT > 0) {
#pragma unroll
      for (int k = 0; k < VPT; ++k) v[k].forget();
    }
  }
  __device__ __forceinline__ float top() const {
    float m = -INFINITY;
    each([&](const Vec<EK>& x, int, int) {
#pragma unroll
      for (int e = 0; e < W; ++e) m = fmaxf(m, x[e]);
    });
    return m;
  }
  // sums of exp((z - m) / tau) and, DUAL, of exp(z - m)
  template <bool DUAL>
  __device__ __forceinline__ void sums(float c, float m, float& s, float& s1) const {
    s = s1 = 0.0f;
    each([&](const Vec<EK>& x, int, int) {
      float p[2] = {0.0f, 0.0f}, p1[2] = {0.0f, 0.0f};
#pragma unroll
      for (int e = 0; e < W; ++e) {
        p[e & 1] += exp_of(x[e], c, m);
        if constexpr (DUAL) p1[e & 1] += exp_of(x[e], kLog2e, m);
      }
      s += p[0] + p[1];
      if constexpr (DUAL) s1 += p1[0] + p1[1];
    });
  }
};

// A row's special classes in LDS: the teacher's, and the label at K (-1: none),
// and -1 behind up to a multiple of 4.
struct Special {
  int* cls;
  float* z;  // their logits
  float* e;  // the teacher's logit; then what the gradient has less there
  int n;     // K + 1, rounded up
};
__device__ __forceinline__ Special special_lds(int K) {
  extern __shared__ __attribute__((aligned(16))) uint8_t dyn[];
  const int n = (K + 4) & ~3;
  return Special{reinterpret_cast<int*>(dyn), reinterpret_cast<float*>(dyn) + n, reinterpret_cast<float*>(dyn) + 2 * n,
                 n};
}
inline unsigned special_bytes(int K) { return (unsigned)((K + 4) & ~3) * 12; }

// Fills cls, z, e of a row; the thread's largest teacher logit.  A term of weight 0
// has no classes: it may be infinite, and 0 inf is NaN.
template <int EK>
__device__ __forceinline__ float gather_special(const DistillArgs& a, int tk, int64_t row, const Special& sp) {
  float tm = -INFINITY;
  const int V = (int)a.V;
  for (int j = threadIdx.x; j < sp.n; j += blockDim.x) {
    int id = -1;
    if (j < a.K) id = a.alpha != 1.0f ? a.ids[row * a.ldi + j] : -1;
    else if (j == a.K && a.labels && a.alpha != 0.0f) id = a.labels[row];
    const bool ok = id >= 0 && id < V;
    sp.cls[j] = ok ? id : -1;
    sp.z[j] = ok ? elem_f32<EK>(a.z, row * a.ldz + id) : 0.0f;
    if (j < a.K) {
      const float x = ok ? elem_any(a.t, row * a.ldt + j, tk) : -INFINITY;
      sp.e[j] = x;
      tm = fmaxf(tm, x);
    } else if (j > a.K) {
      sp.e[j] = 0.0f;
    }
  }
  return tm;
}

// Writes columns [c0, c1) of a row of dz: k2 exp((z - m) / tau) (+ k1 exp(z -
// m)), and the special classes among them with w e less.
template <int EK, bool DUAL, typename P>
__device__ __forceinline__ void write_gradient(const DistillArgs& a, int64_t row, int c0, int c1,
                                               const P& part, const Special& sp, float c2, float m, float k2,
                                               float k1, float w) {
  auto dense = [&](float z) {
    float g = k2 * exp_of(z, c2, m);
    if constexpr (DUAL) g = fmaf(k1, exp_of(z, kLog2e, m), g);
    return g;
  };
  const int hi = part.hi();
  part.each([&](const Vec<EK>& x, int c, int lo) {
    constexpr int W = width(EK);
    float g[W];
#pragma unroll
    for (int e = 0; e < W; ++e) g[e] = dense(x[e]);
    const int64_t at = row * a.lddz + c0 + c;
    if (lo == 0 && hi == W) {
      put_vec<EK, P::STREAM>(a.dz, at, g, W);
    } else {
#pragma unroll
      for (int e = 0; e < W; ++e)
        if (e >= lo && e < hi) put_elem<EK>(a.dz, at + e, g[e]);
    }
  });
  __syncthreads();  // the special classes' dense values are stored
  for (int j = threadIdx.x; j <= a.K; j += blockDim.x) {
    const int id = sp.cls[j];
    if (id < c0 || id >= c1) continue;
    // the same class again: the first of them writes the sum, in the entries' order
    float e = 0.0f;
    bool first = true;
    for (int i = 0; i < sp.n; i += 4) {
      const i32x4_d q = *reinterpret_cast<const i32x4_d*>(sp.cls + i);
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (q[u] == id) {
          e += sp.e[i + u];
          first = first && i + u >= j;
        }
    }
    if (first) put_elem<EK>(a.dz, row * a.lddz + id, dense(sp.z[j]) - w * e);
  }
}

template <int EK, bool STREAM>
__device__ __forceinline__ void write_zeros(const DistillArgs& a, int64_t row, int c0, int c1) {
  constexpr int W = width(EK);
  const float zero[W] = {};
  for (int c = c0 + threadIdx.x * W; c < c1; c += blockDim.x * W) put_vec<EK, STREAM>(a.dz, row * a.lddz + c, zero, c1 - c);
}

// One workgroup a row: 4096 x 32000 bf16 101 us (5.2 TB/s, HBM), 1023 x 50021 f32
// 98 (4.2: a CU holds one row at a time), 1 x 9000 bf16 10 (its chain of loads and
// reductions, and the loss).  The loss alone, with its launch: 4096 x 32000 bf16 53
// (both 106), 1023 x 50021 f32 57 (100).
// Where the row takes at most 32 registers a thread, 8 waves fit a SIMD: a row's
// chain of loads and reductions hides behind other rows'.
template <int NT, int EK, int VPT, bool DUAL>
__global__ __launch_bounds__(NT, VPT * 4 <= 32 && !(DUAL && EK == EL_F32) ? 8 : 4) void distill_row_kernel(DistillArgs a, int tk) {
  const Special sp = special_lds(a.K);
  __shared__ float red[16 * 4];
  constexpr bool STREAM = VPT > 0;
  const int t = threadIdx.x, V = (int)a.V;
  const int64_t row = blockIdx.x;
  const float w = a.w ? a.w[row] : a.w0;
  if (w == 0.0f) {  // left out: not read
    if (a.dz) write_zeros<EK, STREAM>(a, row, 0, V);
    if (t == 0) a.row_loss[row] = 0.0f;
    return;
  }
  const float c2 = a.c2;
  Part<NT, EK, VPT, true, STREAM> part;
  part.open(a.z, row * a.ldz, 0, V);
  float mx[2] = {0.0f, gather_special<EK>(a, tk, row, sp)};
  mx[0] = part.top();
  part.forget();
  block_reduce<0>(mx, red);
  const float m = safe_ref(mx[0]), tm = safe_ref(mx[1]);
  float sm[3];
  part.template sums<DUAL>(c2, m, sm[0], sm[1]);
  part.forget();
  sm[2] = 0.0f;
  for (int j = t; j < a.K; j += blockDim.x) sm[2] += exp_of(sp.e[j], c2, tm);
  block_reduce<1>(sm, red);
  const bool none = mx[0] == -INFINITY;  // no class has any probability
  const float S = none ? __builtin_nanf("") : sm[0], S1 = none ? S : DUAL ? sm[1] : sm[0], ts = sm[2];

  const bool some = !(ts <= 0.0f), has = sp.cls[a.K] >= 0;
  const float soft_w = some ? (1.0f - a.alpha) * a.tau : 0.0f, hard_w = has ? a.alpha : 0.0f;
  const float lgS = log2f(S), lnT = logf(ts), inv_t = some ? 1.0f / ts : 0.0f;
  float l[1] = {0.0f};
  for (int j = t; j < a.K; j += blockDim.x) {
    const float x = (sp.e[j] - tm) / a.tau, p = sp.cls[j] >= 0 ? exp_of(sp.e[j], c2, tm) * inv_t : 0.0f;
    if (p != 0.0f) l[0] += p * ((x - lnT) - ((sp.z[j] - m) * c2 - lgS) * kLn2);
    sp.e[j] = soft_w * p;
  }
  if (t == 0) sp.e[a.K] = hard_w;
  block_reduce<1>(l, red);
  if (t == 0) {
    float rl = (1.0f - a.alpha) * a.tau * a.tau * l[0];
    if (has) rl -= a.alpha * ((sp.z[a.K] - m) - log2f(S1) * kLn2);
    a.row_loss[row] = rl;
  }
  if (!a.dz) return;
  const float k1 = w * hard_w / S1, k2 = w * soft_w / S + (DUAL ? 0.0f : k1);
  write_gradient<EK, DUAL>(a, row, 0, V, part, sp, c2, m, k2, k1, w);
}

// Few rows: P workgroups a row, in two launches.  Each leaves its columns'
// maximum and sums in scratch [R, P, 4]; the first also what the loss takes
// from the teacher and the label (the second launch may write over the logits)
// in the fourth floats: sum p (log p - (z - z0) / tau) in f64, the label's logit,
// and z0, a class's logit, so that nothing large cancels.  8 x 131072 bf16: 5.2 +
// 8.9 us, a load round trip and a few reductions each.
constexpr int kPartNT = 256;
__device__ __forceinline__ void part_columns(int V, int P, int* c0, int* c1) {
  const int len = ((V + P - 1) / P + 7) & ~7;
  *c0 = min((int)blockIdx.x * len, V);
  *c1 = min(*c0 + len, V);
}

template <int EK, int VPT, bool DUAL>
__global__ __launch_bounds__(kPartNT) void distill_stats_kernel(DistillArgs a, int tk, float* scratch, int P, int ldp) {
  const Special sp = special_lds(a.K);
  __shared__ float red[kPartNT / 64 * 4];
  __shared__ double red64[kPartNT / 64];
  __shared__ float z0s;
  const int64_t row = blockIdx.y;
  const float w = a.w ? a.w[row] : a.w0;
  if (w == 0.0f) return;
  int c0, c1;
  part_columns((int)a.V, P, &c0, &c1);
  const float c2 = a.c2;
  Part<kPartNT, EK, VPT, false, false> part;
  part.open(a.z, row * a.ldz, c0, c1);
  float mx[1] = {part.top()};
  block_reduce<0>(mx, red);
  float sm[2];
  part.template sums<DUAL>(c2, safe_ref(mx[0]), sm[0], sm[1]);
  block_reduce<1>(sm, red);
  float* out = scratch + (row * ldp + blockIdx.x) * 4;
  if (threadIdx.x == 0) {
    out[0] = mx[0];
    out[1] = sm[0];
    out[2] = sm[1];
  }
  if (blockIdx.x != 0) return;
  float tm[1] = {gather_special<EK>(a, tk, row, sp)};
  block_reduce<0>(tm, red);
  tm[0] = safe_ref(tm[0]);
  if (threadIdx.x == 0) {
    int j = 0;
    while (j < a.K && sp.cls[j] < 0) ++j;
    const float z = j < a.K ? sp.z[j] : 0.0f;
    z0s = fabsf(z) < INFINITY ? z : 0.0f;
  }
  float ts[1] = {0.0f};
  for (int j = threadIdx.x; j < a.K; j += blockDim.x) ts[0] += exp_of(sp.e[j], c2, tm[0]);
  block_reduce<1>(ts, red);
  const double c2e = (double)c2 * 0.6931471805599453;  // as the sums' exponentials have it
  const float lnT = logf(ts[0]), inv_t = !(ts[0] <= 0.0f) ? 1.0f / ts[0] : 0.0f;
  double l = 0.0;
  for (int j = threadIdx.x; j < a.K; j += blockDim.x) {
    const float x = (sp.e[j] - tm[0]) / a.tau, p = sp.cls[j] >= 0 ? exp_of(sp.e[j], c2, tm[0]) * inv_t : 0.0f;
    if (p != 0.0f) l += (double)p * ((double)(x - lnT) - ((double)sp.z[j] - (double)z0s) * c2e);
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) l += __shfl_xor(l, off, 64);
  if ((threadIdx.x & 63) == 0) red64[threadIdx.x >> 6] = l;
  __syncthreads();
  if (threadIdx.x == 0) {
    l = (red64[0] + red64[1]) + (red64[2] + red64[3]);
    const uint64_t bits = (uint64_t)__double_as_longlong(l);
    out[3] = __uint_as_float((uint32_t)bits);
    out[7] = __uint_as_float((uint32_t)(bits >> 32));
    out[11] = sp.z[a.K];
    out[15] = z0s;
  }
}

template <int EK, int VPT, bool DUAL>
__global__ __launch_bounds__(kPartNT) void distill_grad_kernel(DistillArgs a, int tk, const float* scratch, int P,
                                                               int ldp) {
  const Special sp = special_lds(a.K);
  __shared__ float red[kPartNT / 64 * 4];
  const int64_t row = blockIdx.y;
  const int t = threadIdx.x;
  const float w = a.w ? a.w[row] : a.w0;
  int c0, c1;
  part_columns((int)a.V, P, &c0, &c1);
  if (w == 0.0f) {
    if (a.dz) write_zeros<EK, false>(a, row, c0, c1);
    if (t == 0 && blockIdx.x == 0) a.row_loss[row] = 0.0f;
    return;
  }
  const float c2 = a.c2;
  Part<kPartNT, EK, VPT, false, false> part;
  if (a.dz) part.open(a.z, row * a.ldz, c0, c1);
  // the row's statistics, and the special classes: those of other
  // workgroups' columns only for their probabilities, as their logits may be written over by now
  const float* in = scratch + row * ldp * 4;
  f32x4 own = {-INFINITY, 0.0f, 0.0f, 0.0f};  // P <= 64: one a lane, the same in every wave
  if ((t & 63) < P) own = *reinterpret_cast<const f32x4_a4*>(in + (t & 63) * 4);
  // (a part without a class, and a lane without a part, has the maximum -inf and the factor 0: with 0 in the
  // maximum's place the factor would overflow far below zero, and 0 inf is NaN)
  const float mx = wave_max(own[0]), m = safe_ref(mx);
  float S = wave_sum(own[1] * exp_of(own[0], c2, m));
  float S1 = DUAL ? wave_sum(own[2] * exp_of(own[0], kLog2e, m)) : S;
  if (mx == -INFINITY) S = S1 = __builtin_nanf("");
  float tm[1] = {gather_special<EK>(a, tk, row, sp)};
  block_reduce<0>(tm, red);
  tm[0] = safe_ref(tm[0]);
  float ts[1] = {0.0f};
  for (int j = t; j < a.K; j += blockDim.x) ts[0] += exp_of(sp.e[j], c2, tm[0]);
  block_reduce<1>(ts, red);
  const bool some = !(ts[0] <= 0.0f), has = sp.cls[a.K] >= 0;
  const float soft_w = some ? (1.0f - a.alpha) * a.tau : 0.0f, hard_w = has ? a.alpha : 0.0f;
  const float inv_t = some ? 1.0f / ts[0] : 0.0f;
  float pr[1] = {0.0f};  // the sum of the probabilities: 1, or 0 without a teacher, or NaN
  for (int j = t; j < a.K; j += blockDim.x) {
    const float p = sp.cls[j] >= 0 ? exp_of(sp.e[j], c2, tm[0]) * inv_t : 0.0f;
    pr[0] += p;
    sp.e[j] = soft_w * p;
  }
  if (t == 0) sp.e[a.K] = hard_w;
  block_reduce<1>(pr, red);
  if (t == 0 && blockIdx.x == 0) {
    const double l = __longlong_as_double((long long)((uint64_t)__float_as_uint(in[3]) |
                                                      (uint64_t)__float_as_uint(in[7]) << 32));
    // sum p (log p - (z - z0) / tau) + sum p (log sum exp(z / tau) - z0 / tau)
    const double lse = (((double)m - (double)in[15]) * (double)c2 + (double)log2f(S)) * 0.6931471805599453;
    float rl = some ? (1.0f - a.alpha) * a.tau * a.tau * (float)(l + (double)pr[0] * lse) : 0.0f;
    if (has) rl -= a.alpha * ((in[11] - m) - log2f(S1) * kLn2);
    a.row_loss[row] = rl;
  }
  if (!a.dz) return;
  const float k1 = w * hard_w / S1, k2 = w * soft_w / S + (DUAL ? 0.0f : k1);
  write_gradient<EK, DUAL>(a, row, c0, c1, part, sp, c2, m, k2, k1, w);
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
  // tau^2 and log2(e) / tau stay within f32's range
  if (!(c.tau >= 0x1p-60f && c.tau <= 0x1p60f) || !(c.alpha >= 0.0f && c.alpha <= 1.0f)) return false;
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
  if (R < 1 || V < 1 || R > INT32_MAX || V > (1 << 28)) return false;  // a row's byte offsets: 32 bits
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

// Row r of the tensors becomes the first.
template <int EK>
DistillArgs from_row(const DistillArgs& a, int tk, int64_t r, int64_t rows) {
  const int64_t es = EK == EL_F32 ? 4 : 2, et = tk == EL_F32 ? 4 : 2;
  DistillArgs p = a;
  p.R = rows;
  p.z = (const uint8_t*)a.z + r * a.ldz * es;
  p.t = (const uint8_t*)a.t + r * a.ldt * et;
  p.ids = a.ids + r * a.ldi;
  if (a.labels) p.labels = a.labels + r;
  if (a.w) p.w = a.w + r;
  if (a.dz) p.dz = (uint8_t*)a.dz + r * a.lddz * es;
  p.row_loss = a.row_loss + r;
  return p;
}

template <int EK, bool DUAL>
Status distill_rows(const DistillArgs& a, int tk, float* scratch, int ldp, hipStream_t s) {
  // Few long rows share the chip: parts of 2048 columns or more, about two
  // workgroups a CU.  A row a workgroup against this: 8 x 200000 bf16 37.9 us
  // (17.1), 8 x 65536 19.4 (16.6), f32 22.2 (16.3), 48 x 131072 28.2 (24.9); the
  // other way 8 x 32000 f32 12.8 (15.1), 128 x 131072 f32 45.8 (51.3).
  const unsigned lds = special_bytes(a.K);
  int64_t P = (512 + a.R - 1) / a.R;
  if (P > a.V / 2048) P = a.V / 2048;
  if (P > ldp) P = ldp;
  if (P > 64) P = 64;
  if (scratch && a.R <= 48 && a.V >= 49152 && P >= 4) {  // (a row's last words are in the fourth part's floats)
    const dim3 grid((unsigned)P, (unsigned)a.R);
    const int64_t len = (a.V + P - 1) / P + 7;
    auto go = [&](auto vpt) {
      constexpr int VPT = decltype(vpt)::value;
      distill_stats_kernel<EK, VPT, DUAL><<<grid, kPartNT, lds, s>>>(a, tk, scratch, (int)P, ldp);
      distill_grad_kernel<EK, VPT, DUAL><<<grid, kPartNT, lds, s>>>(a, tk, scratch, (int)P, ldp);
    };
    if (len <= kPartNT * 8 * 2) go(std::integral_constant<int, 2 * 8 / width(EK)>{});
    else go(std::integral_constant<int, 0>{});
    return launch_status("distill_topk");
  }
  // The row in the registers of the fewest threads that hold it: up to 64
  // columns a thread in 16 bits and 56 in f32 (128 in 16 bits for the longest);
  // beyond 2^17 or 57344 columns it is read in each pass.
  const int64_t kStep = 1 << 21;  // rows a launch: a grid's lanes are counted in 32 bits
  for (int64_t r = 0; r < a.R; r += kStep) {
    const DistillArgs p = from_row<EK>(a, tk, r, a.R - r < kStep ? a.R - r : kStep);
    const unsigned g = (unsigned)p.R;
    constexpr int L = EK == EL_F32 ? 7 : 8, XL = EK == EL_F32 ? 0 : 16;
#define DISTILL_ROW(NT, VPT)                                                                  \
  do {                                                                                        \
    constexpr int N = (VPT) * 8 / width(EK);                                                  \
    distill_row_kernel<NT, EK, N, DUAL><<<g, NT, lds, s>>>(p, tk);                            \
  } while (0)
    if (a.V <= 512) DISTILL_ROW(64, 1);
    else if (a.V <= 1024) DISTILL_ROW(64, 2);
    else if (a.V <= 2048) DISTILL_ROW(64, 4);
    else if (a.V <= 4096) DISTILL_ROW(128, 4);
    else if (a.V <= 8192) DISTILL_ROW(256, 4);
    else if (a.V <= 16384) DISTILL_ROW(512, 4);
    else if (a.V <= 512 * 8 * L) DISTILL_ROW(512, L);
    else if (a.V <= 1024 * 8 * L) DISTILL_ROW(1024, L);
    else if (XL && a.V <= 131072) DISTILL_ROW(1024, XL);
    else distill_row_kernel<1024, EK, 0, DUAL><<<g, 1024, lds, s>>>(p, tk);
#undef DISTILL_ROW
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
  a.c2 = (float)(1.4426950408889634 / (double)c.tau);
  int ek, tk;
  elem_kind(*c.z, &ek);
  elem_kind(*c.t, &tk);
  hipStream_t s = as_stream(stream);
  const bool dual = a.labels && a.alpha != 0.0f && a.tau != 1.0f;
  float* sc = c.scratch ? (float*)c.scratch->data : nullptr;
  const int ldp = c.scratch ? (int)c.scratch->shape[1] : 0;
  Status st;
  if (ek == EL_F32)
    st = dual ? distill_rows<EL_F32, true>(a, tk, sc, ldp, s) : distill_rows<EL_F32, false>(a, tk, sc, ldp, s);
  else if (ek == EL_F16)
    st = dual ? distill_rows<EL_F16, true>(a, tk, sc, ldp, s) : distill_rows<EL_F16, false>(a, tk, sc, ldp, s);
  else
    st = dual ? distill_rows<EL_BF16, true>(a, tk, sc, ldp, s) : distill_rows<EL_BF16, false>(a, tk, sc, ldp, s);
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
