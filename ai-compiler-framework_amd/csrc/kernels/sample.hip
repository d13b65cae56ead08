// One draw a row from given random numbers, with temperature, top-k, top-p and
// min-p of each row's own.
//
//   order   falling logit, equal logits by rising class; as one integer, the
//           order's composite (~key << 32 | class) rises along it
//   w       exp((z - max) / T), held as whole numbers of 2^-S
//   top-k   the first k of the order
//   top-p   of those, the ones before which w adds up to less than top_p W
//   min-p   of those, the ones with w >= min_p
//   token   the lowest class at which the sum of the kept w, taken over the
//           classes in their own order, passes u W
//
// Every cut is a prefix of the order, so what is kept is "composite <= limit"
// (and w >= min_p).  A limit is found by a histogram of the row, its one bin
// that holds the cut, and a sort of that bin's members (or of everything above
// it, where that is little).
//
// A sum's rounding draws another token, so no sum is rounded: w is computed in
// f64 and rounded once to a multiple of 2^-S, and the sums are 64-bit integers,
// the same whatever the order of their terms, LDS atomics among them.  S = 62 -
// ceil(log2 V), at most 51: for 2^17 classes a term is off by at most 2^-46 of
// the largest weight.
//
// A workgroup owns a row and reads it again, from the caches, in each pass.
//
// No counterpart in the reference.
#include "../common/head_util.hpp"

namespace aicf::hip {

namespace {

typedef unsigned long long u64;

struct SampleArgs {
  const void* z;
  const float* u;
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  int32_t* token;
  float* logprob;  // may be nullptr
  int64_t ldz;
  int R, V, shift;  // shift: S
};

constexpr int kBins = 1536;  // of 1 + distance / T: 256 an octave, 6 octaves; the last takes all beyond
constexpr int kList = 2048;  // members a limit is sorted out of

// exp(-y) 2^S for y >= 0, to the nearest integer: 2^t = 2^n 2^f with |f| <=
// 1/2, the series of 2^f to f^11 (1e-14 relative).
__device__ __forceinline__ u64 weight_of(double y, int S) {
  y = fmin(y, 800.0);
  const double t = -y * 1.4426950408889634, n = rint(t), f = (t - n) * 0.6931471805599453;
  double p = 1.0 / 39916800.0;
  p = fma(p, f, 1.0 / 3628800.0);
  p = fma(p, f, 1.0 / 362880.0);
  p = fma(p, f, 1.0 / 40320.0);
  p = fma(p, f, 1.0 / 5040.0);
  p = fma(p, f, 1.0 / 720.0);
  p = fma(p, f, 1.0 / 120.0);
  p = fma(p, f, 1.0 / 24.0);
  p = fma(p, f, 1.0 / 6.0);
  p = fma(p, f, 0.5);
  p = fma(p, f, 1.0);
  p = fma(p, f, 1.0);
  // adding 2^52 leaves the integer in the low bits
  const double r = ldexp(p, (int)n + S) + 4503599627370496.0;
  return (u64)__double_as_longlong(r) - 0x4330000000000000ull;
}

__device__ __forceinline__ uint32_t key_of(float z) {
  const uint32_t b = __float_as_uint(z);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
constexpr uint32_t kKeyNone = 0x007fffffu;  // the key of -inf
__device__ __forceinline__ float z_of_key(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
// A logit as the order sees it: NaN is -inf, -0 is 0.
__device__ __forceinline__ float clean(float z) { return z == z ? z + 0.0f : -INFINITY; }

__device__ __forceinline__ u64 shfl_xor64(u64 v, int off) { return (u64)__shfl_xor((long long)v, off, 64); }
__device__ __forceinline__ u64 shfl_up64(u64 v, int off) { return (u64)__shfl_up((long long)v, off, 64); }
__device__ __forceinline__ u64 wave_sum64(u64 v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += shfl_xor64(v, off);
  return v;
}
__device__ __forceinline__ u64 wave_scan64(u64 v) {  // inclusive
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const u64 o = shfl_up64(v, off);
    if (lane >= off) v += o;
  }
  return v;
}

template <int NT>
struct SampleLds {
  uint32_t cnt[kBins];
  u64 mass[kBins];
  u64 list[kList];
  u64 wred[NT / 64 + 1], wred2[NT / 64 + 1];
  u64 b64[4];
  int bi[4];
};

template <int EK, int NT>
struct SampleRow {
  static constexpr int NW = NT / 64;

  const SampleArgs& a;
  SampleLds<NT>& s;
  const uint8_t* z;  // the row
  int nvec;          // vectors of 8 a thread
  float zmax;
  double inv_t;
  float inv_tf;

  // The thread's vector k: classes (k NT + t) 8 .. +7; past the row: -inf.
  __device__ __forceinline__ int first(int k) const { return (k * NT + (int)threadIdx.x) * 8; }
  __device__ __forceinline__ void get(int k, float (&v)[8]) const {
    const int c = first(k), n = a.V - c;
    load8<EK>(v, z, c, n);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < n ? clean(v[e]) : -INFINITY;
  }
  // f(z, class) for every element of the thread
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    for (int k = 0; k < nvec; ++k) {
      float v[8];
      get(k, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) f(v[e], first(k) + e);
    }
  }

  __device__ __forceinline__ u64 weight(float v) const {
    if (v == zmax) return 1ull << a.shift;
    return weight_of(((double)zmax - (double)v) * inv_t, a.shift);
  }
  __device__ __forceinline__ static u64 comp(float v, int c) { return ((u64)(~key_of(v)) << 32) | (uint32_t)c; }
  __device__ __forceinline__ int bin_of(float v) const {
    // rounding is monotone: a lower logit never has a lower bin
    const float y = v == zmax ? 1.0f : fmaf(zmax - v, inv_tf, 1.0f);
    const int b = (int)((__float_as_uint(y) >> 15) - (0x3f800000u >> 15));
    return y < 64.0f ? b : kBins - 1;  // (not <: beyond, or NaN)
  }

  // block reductions; the result in every thread
  __device__ __forceinline__ u64 block_min64(u64 v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
      const u64 o = shfl_xor64(v, off);
      v = o < v ? o : v;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s.wred[threadIdx.x >> 6] = v;
    __syncthreads();
    v = s.wred[0];
#pragma unroll
    for (int k = 1; k < NW; ++k) v = s.wred[k] < v ? s.wred[k] : v;
    return v;
  }
  __device__ __forceinline__ u64 block_sum64(u64 v) {
    v = wave_sum64(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s.wred[threadIdx.x >> 6] = v;
    __syncthreads();
    v = s.wred[0];
#pragma unroll
    for (int k = 1; k < NW; ++k) v += s.wred[k];
    return v;
  }

  __device__ __forceinline__ void clear_hist(int bins) {
    __syncthreads();
    for (int i = threadIdx.x; i < bins; i += NT) {
      s.cnt[i] = 0;
      s.mass[i] = 0;
    }
    __syncthreads();
  }

  // The first of `bins` bins up to which the counts (or masses) reach target;
  // -> bin, its count, and what lies before it.  The last bin if none does.
  struct Cut {
    int bin;
    uint32_t n, cnt_before;
    u64 mass_before;
  };
  __device__ __forceinline__ Cut find_bin(int bins, bool by_mass, u64 target) {
    __syncthreads();
    const int per = (bins + NT - 1) / NT, b0 = threadIdx.x * per;
    u64 c = 0, m = 0;
    for (int i = b0; i < b0 + per && i < bins; ++i) {
      c += s.cnt[i];
      m += s.mass[i];
    }
    const u64 ci = wave_scan64(c), mi = wave_scan64(m);
    if ((threadIdx.x & 63) == 63) {
      s.wred[threadIdx.x >> 6] = ci;
      s.wred2[threadIdx.x >> 6] = mi;
    }
    if (threadIdx.x == 0) s.bi[0] = -1;
    __syncthreads();
    u64 cb = ci - c, mb = mi - m, call = 0, mall = 0;
    for (int k = 0; k < NW; ++k) {
      if (k < (int)(threadIdx.x >> 6)) {
        cb += s.wred[k];
        mb += s.wred2[k];
      }
      call += s.wred[k];
      mall += s.wred2[k];
    }
    const u64 want = min(target, by_mass ? mall : call);
    // one thread's range holds the crossing: before < want <= before + own
    if ((by_mass ? mb : cb) < want && want <= (by_mass ? mb + m : cb + c)) {
      for (int i = b0; i < b0 + per && i < bins; ++i) {
        const u64 own = by_mass ? s.mass[i] : s.cnt[i];
        if ((by_mass ? mb : cb) + own >= want) {
          s.bi[0] = i;
          s.bi[1] = (int)s.cnt[i];
          s.b64[0] = cb;
          s.b64[1] = mb;
          break;
        }
        cb += s.cnt[i];
        mb += s.mass[i];
      }
    }
    __syncthreads();
    return Cut{s.bi[0], (uint32_t)s.bi[1], (uint32_t)s.b64[0], s.b64[1]};
  }

  // Sorts list[0 .. n) rising; n <= kList.
  __device__ __forceinline__ void sort_list(int n) {
    int m = 64;
    while (m < n) m <<= 1;
    __syncthreads();
    for (int i = n + threadIdx.x; i < m; i += NT) s.list[i] = ~0ull;
    for (int k = 2; k <= m; k <<= 1)
      for (int j = k >> 1; j > 0; j >>= 1) {
        __syncthreads();
        for (int q = threadIdx.x; q < m / 2; q += NT) {
          const int i = (q / j) * 2 * j + q % j, o = i + j;
          const u64 x = s.list[i], y = s.list[o];
          if ((x > y) == ((i & k) == 0)) {
            s.list[i] = y;
            s.list[o] = x;
          }
        }
      }
    __syncthreads();
  }

  // The last entry of the sorted list[0 .. n) before which, `before` included,
  // the masses add up to less than target; its index.
  __device__ __forceinline__ int last_below(int n, u64 before, u64 target) {
    constexpr int PER = kList / NT > 0 ? kList / NT : 1;
    u64 w[PER], own = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int j = threadIdx.x * PER + i;
      w[i] = j < n ? weight(z_of_key(~(uint32_t)(s.list[j] >> 32))) : 0;
      own += w[i];
    }
    u64 run = wave_scan64(own) - own;
    if ((threadIdx.x & 63) == 63) s.wred[threadIdx.x >> 6] = run + own;
    if (threadIdx.x == 0) s.bi[2] = 0;
    __syncthreads();
    for (int k = 0; k < (int)(threadIdx.x >> 6); ++k) run += s.wred[k];
    run += before;
    int last = -1;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int j = threadIdx.x * PER + i;
      if (j < n && run < target) last = j;
      run += w[i];
    }
    if (last >= 0) atomicMax(&s.bi[2], last);
    __syncthreads();
    return s.bi[2];
  }

  // Fills list with the composites of the elements f accepts.
  template <typename F>
  __device__ __forceinline__ int compact(F f) {
    __syncthreads();
    if (threadIdx.x == 0) s.bi[3] = 0;
    __syncthreads();
    each([&](float v, int c) {
      if (f(v, c)) {
        const int at = atomicAdd(&s.bi[3], 1);
        if (at < kList) s.list[at] = comp(v, c);
      }
    });
    __syncthreads();
    return s.bi[3];
  }

  // Among the elements with composite <= limit: the composite of the target-th
  // (by count), or of the last one before which the masses add up to less than
  // target.  `cut` is the bin of bin_of that holds it.
  __device__ u64 refine(u64 limit, bool by_mass, u64 target, Cut cut) {
    // the bin's members span composites [lo, hi]
    u64 lo = ~0ull, hi_inv = ~0ull;
    const int b0 = cut.bin;
    each([&](float v, int c) {
      const u64 q = comp(v, c);
      if (key_of(v) > kKeyNone && q <= limit && bin_of(v) == b0) {
        lo = q < lo ? q : lo;
        hi_inv = ~q < hi_inv ? ~q : hi_inv;
      }
    });
    lo = block_min64(lo);
    u64 hi = ~block_min64(hi_inv);
    u64 cnt_before = cut.cnt_before, mass_before = cut.mass_before;
    u64 n = cut.n;
    while (n > kList) {
      // 1024 bins over [lo, hi]
      int shift = 64 - __clzll((long long)(hi - lo)) - 10;
      shift = shift < 0 ? 0 : shift;
      clear_hist(1024);
      each([&](float v, int c) {
        const u64 q = comp(v, c);
        if (q >= lo && q <= hi) {
          const int b = (int)((q - lo) >> shift);
          atomicAdd(&s.cnt[b], 1u);
          if (by_mass) atomicAdd(&s.mass[b], weight(v));
        }
      });
      const Cut k = find_bin(1024, by_mass, target - (by_mass ? mass_before : cnt_before));
      cnt_before += k.cnt_before;
      mass_before += k.mass_before;
      n = k.n;
      const u64 base = lo + ((u64)k.bin << shift), top = base + ((1ull << shift) - 1);
      lo = base;
      hi = top < hi ? top : hi;
    }
    const int m = compact([&](float v, int c) {
      const u64 q = comp(v, c);
      return q >= lo && q <= hi;
    });
    sort_list(m);
    int at;
    if (by_mass) {
      at = last_below(m, mass_before, target);
    } else {
      at = (int)(target - cnt_before) - 1;
      at = at < m ? at : m - 1;
    }
    const u64 q = s.list[at];
    __syncthreads();
    return q;
  }

  __device__ __forceinline__ void write(int token, float lp) const {
    if (threadIdx.x == 0) {
      a.token[blockIdx.x] = token;
      if (a.logprob) a.logprob[blockIdx.x] = lp;
    }
  }
  __device__ __forceinline__ float log_of(float v, u64 total) const {
    const double d = v == zmax ? 0.0 : ((double)zmax - (double)v) * inv_t;
    return (float)(-d - log(ldexp((double)total, -a.shift)));
  }
  __device__ __forceinline__ u64 draw_at(u64 total) const {
    float u = a.u[blockIdx.x];
    u = u > 0.0f ? fminf(u, 0.99999994f) : 0.0f;
    return (u64)((double)u * (double)total);  // the sum has to pass this
  }

  // The draw where everything kept is in list[0 .. m), sorted by composite.
  __device__ void draw_small(int m) {
    // into the order of the classes, the key in the low half
    for (int i = threadIdx.x; i < m; i += NT) s.list[i] = (s.list[i] << 32) | (s.list[i] >> 32);
    sort_list(m);
    constexpr int PER = kList / NT > 0 ? kList / NT : 1;
    u64 w[PER], own = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int j = threadIdx.x * PER + i;
      w[i] = j < m ? weight(z_of_key(~(uint32_t)s.list[j])) : 0;
      own += w[i];
    }
    u64 run = wave_scan64(own) - own;
    if ((threadIdx.x & 63) == 63) s.wred[threadIdx.x >> 6] = run + own;
    __syncthreads();
    u64 total = 0;
    for (int k = 0; k < NW; ++k) {
      if (k < (int)(threadIdx.x >> 6)) run += s.wred[k];
      total += s.wred[k];
    }
    const u64 at = draw_at(total);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (run <= at && at < run + w[i]) {
        const u64 q = s.list[threadIdx.x * PER + i];
        a.token[blockIdx.x] = (int)(q >> 32);
        if (a.logprob) a.logprob[blockIdx.x] = log_of(z_of_key(~(uint32_t)q), total);
      }
      run += w[i];
    }
  }

  // The draw over the row: kept are composites <= limit with weight >= least.
  __device__ void draw_row(u64 limit, u64 least) {
    auto kept = [&](float v, int c) -> u64 {
      if (key_of(v) <= kKeyNone || comp(v, c) > limit) return 0;
      const u64 w = weight(v);
      return w >= least ? w : 0;
    };
    u64 own = 0;
    each([&](float v, int c) { own += kept(v, c); });
    const u64 total = block_sum64(own), at = draw_at(total);
    // segments of 512 classes (a vector of a wave) in the order of the classes
    u64 before = 0;
    for (int k = 0; k < nvec; ++k) {
      float v[8];
      get(k, v);
      u64 w[8], sum = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        w[e] = kept(v[e], first(k) + e);
        sum += w[e];
      }
      const u64 incl = wave_scan64(sum);
      __syncthreads();
      if ((threadIdx.x & 63) == 63) s.wred[threadIdx.x >> 6] = incl;
      __syncthreads();
      u64 run = before + incl - sum;
      for (int q = 0; q < NW; ++q) {
        if (q < (int)(threadIdx.x >> 6)) run += s.wred[q];
        before += s.wred[q];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (run <= at && at < run + w[e]) {
          a.token[blockIdx.x] = first(k) + e;
          if (a.logprob) a.logprob[blockIdx.x] = log_of(v[e], total);
        }
        run += w[e];
      }
      if (before > at) return;
    }
  }

  __device__ void run() {
    const int row = blockIdx.x;
    const float T = a.temperature[row], top_p = a.top_p[row], min_p = a.min_p[row];
    const int top_k = a.top_k[row];
    nvec = (a.V + NT * 8 - 1) / (NT * 8);
    u64 best = ~0ull;
    each([&](float v, int c) {
      const u64 q = comp(v, c);
      best = q < best ? q : best;
    });
    best = block_min64(best);
    zmax = z_of_key(~(uint32_t)(best >> 32));
    if (zmax == -INFINITY) return write(-1, -INFINITY);
    if (!(T > 0.0f) || top_k == 1 || top_p <= 0.0f) return write((int)(uint32_t)best, 0.0f);
    inv_t = 1.0 / (double)T;
    inv_tf = (float)inv_t;
    u64 least = 0;
    // w >= min_p: on the rounded weights, the least whole number that min_p admits
    if (min_p > 0.0f) least = (u64)ceil(ldexp((double)fminf(min_p, 1.0f), a.shift));
    const bool by_k = top_k > 0 && top_k < a.V, by_p = top_p < 1.0f;
    u64 limit = ~0ull;
    for (int pass = 0; pass < 2; ++pass) {
      const bool by_mass = pass == 1;
      if (!(by_mass ? by_p : by_k)) continue;
      clear_hist(kBins);
      each([&](float v, int c) {
        if (key_of(v) > kKeyNone && comp(v, c) <= limit) {
          const int b = bin_of(v);
          atomicAdd(&s.cnt[b], 1u);
          if (by_mass) atomicAdd(&s.mass[b], weight(v));
        }
      });
      u64 target = (u64)top_k;
      if (by_mass) {
        u64 own = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < kBins; i += NT) own += s.mass[i];
        target = (u64)ceil((double)top_p * (double)block_sum64(own));
      }
      const Cut cut = find_bin(kBins, by_mass, target);
      if (cut.cnt_before + cut.n <= kList) {
        // little lies up to the cut: all of it, sorted
        int m = compact([&](float v, int c) {
          return key_of(v) > kKeyNone && comp(v, c) <= limit && bin_of(v) <= cut.bin;
        });
        sort_list(m);
        if (!by_mass) {
          m = top_k < m ? top_k : m;
          if (by_p) {
            constexpr int PER = kList / NT > 0 ? kList / NT : 1;
            u64 own = 0;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
              const int j = threadIdx.x * PER + i;
              if (j < m) own += weight(z_of_key(~(uint32_t)(s.list[j] >> 32)));
            }
            const u64 total = block_sum64(own);
            __syncthreads();
            m = last_below(m, 0, (u64)ceil((double)top_p * (double)total)) + 1;
          }
        } else {
          m = last_below(m, 0, target) + 1;
        }
        if (least) {  // the weights fall along the order
          int n = 0;
          for (int j = threadIdx.x; j < m; j += NT)
            if (weight(z_of_key(~(uint32_t)(s.list[j] >> 32))) >= least) ++n;
          m = (int)block_sum64((u64)n);
        }
        __syncthreads();
        return draw_small(m);
      }
      limit = refine(limit, by_mass, target, cut);
    }
    draw_row(limit, least);
  }
};

template <int EK, int NT>
__global__ __launch_bounds__(NT) void sample_kernel(SampleArgs a) {
  __shared__ SampleLds<NT> lds;
  SampleRow<EK, NT> row{a, lds,
                             static_cast<const uint8_t*>(a.z) + (int64_t)blockIdx.x * a.ldz * (EK == EL_F32 ? 4 : 2)};
  row.run();
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
bool sample_sup(const TensorDesc* in, int ni, const TensorDesc* out, int no, const void*) {
  if (!in || !out || ni != 6 || no < 1 || no > 3) return false;
  int ek;
  int64_t ld;
  if (!elem_kind(in[0], &ek) || !matrix_ld(in[0], false, &ld)) return false;
  const int64_t R = in[0].shape[0], V = in[0].shape[1];
  if (V < 1 || V > (1 << 24) || R > (1 << 21)) return false;
  for (int i = 1; i < 6; ++i)
    if (!vector_of(in[i], i == 3 ? DType::kI32 : DType::kF32, R)) return false;
  if (!vector_of(out[0], DType::kI32, R)) return false;
  if (no > 1 && !vector_of(out[1], DType::kF32, R)) return false;
  if (no > 2) {
    const TensorDesc& s = out[2];
    if (dt(s) != DType::kI32 || !s.contiguous || s.rank != 2 || s.shape[0] != R || s.shape[1] < 8192) return false;
  }
  return !any_overlap(in, ni, out, no);
}

template <int EK>
Status sample_run(const SampleArgs& a, hipStream_t s) {
  const unsigned g = (unsigned)a.R;
  if (a.V <= 8192) sample_kernel<EK, 256><<<g, 256, 0, s>>>(a);
  else sample_kernel<EK, 1024><<<g, 1024, 0, s>>>(a);
  return launch_status("sample_row");
}

Status sample_launch(const TensorDesc* in, int ni, TensorDesc* out, int no, const void* at, void*, size_t,
                     void* stream) {
  if (!sample_sup(in, ni, out, no, at)) return Status::InvalidArgument;
  if (in[0].shape[0] == 0) return Status::Ok;
  for (int k = 0; k < ni; ++k)
    if (no_memory(in[k])) return Status::InvalidArgument;
  for (int k = 0; k < no; ++k)
    if (no_memory(out[k])) return Status::InvalidArgument;
  SampleArgs a{};
  a.R = (int)in[0].shape[0];
  a.V = (int)in[0].shape[1];
  a.z = in[0].data;
  matrix_ld(in[0], false, &a.ldz);
  a.u = (const float*)in[1].data;
  a.temperature = (const float*)in[2].data;
  a.top_k = (const int32_t*)in[3].data;
  a.top_p = (const float*)in[4].data;
  a.min_p = (const float*)in[5].data;
  a.token = (int32_t*)out[0].data;
  a.logprob = no > 1 ? (float*)out[1].data : nullptr;
  int bits = 0;
  while ((int64_t{1} << bits) < a.V) ++bits;
  a.shift = 62 - bits < 51 ? 62 - bits : 51;
  int ek;
  elem_kind(in[0], &ek);
  hipStream_t s = as_stream(stream);
  if (ek == EL_F32) return sample_run<EL_F32>(a, s);
  return ek == EL_F16 ? sample_run<EL_F16>(a, s) : sample_run<EL_BF16>(a, s);
}

size_t no_workspace(const TensorDesc*, int, const void*) { return 0; }

}  // namespace

KernelVariant make_sample_row_variant() {
  KernelVariant v;
  v.name = "sample_row";
  v.launch = sample_launch;
  v.supported = sample_sup;
  v.query_workspace = no_workspace;
  return v;
}

}  // namespace aicf::hip
