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
// (and w >= min_p).  A limit is found by a histogram of the row, finer ones of
// the bin that holds the cut, and the order of the last few by counting; where
// little lies up to the cut, that alone is ordered and drawn from.
//
// A sum's rounding draws another token, so no sum is rounded: w is computed in
// f64 and rounded once to a multiple of 2^-S, and the sums are 64-bit integers,
// the same whatever the order of their terms, LDS atomics among them.  S = 62 -
// ceil(log2 V), at most 51: for 2^17 classes a term is off by at most 2^-46 of
// the largest weight.
//
// A workgroup owns a row and reads it again, from the caches, in each pass.  256
// x 65521 bf16: greedy 12-15 us, top-k 50 30, plain draws 41, top-p 0.9 100; the
// f64 weights (half rate, some 20 operations each) and the histogram's 64-bit LDS
// atomics bound them, not the 7 us of bytes.
//
// No counterpart in the reference.
#include "../common/head_util.hpp"

namespace aicf::hip {

namespace {

typedef unsigned long long u64;
typedef uint32_t u32x4_a2 __attribute__((ext_vector_type(4), aligned(2)));

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

// 2^(S - t) for t >= 0, to the nearest integer: 2^n 2^f with |f| <= 1/2, the
// series of 2^f to f^10 (at most 2.2e-13 off, relative).  Adding 1.5 2^52 rounds
// t to an integer in the sum's low bits, adding to the exponent field scales,
// adding 2^52 leaves the rounded result in the low bits: conversions and ldexp
// issue at a quarter of the rate of f64 additions.
// The series' coefficients stay in scalar registers: as literals each would be
// moved to a vector register for every term.
struct Exp2Series {
  double k[11];
  __device__ __forceinline__ Exp2Series() {
    constexpr double L = 0.6931471805599453;
    double c = 1.0;
#pragma unroll
    for (int i = 0; i < 11; ++i) {
      k[i] = c;
      asm volatile("" : "+s"(k[i]));
      c *= L / (i + 1);
    }
  }
};
__device__ __forceinline__ u64 weight_of(const Exp2Series& x, double t, int S) {
  t = fmin(t, 900.0);
  const double r = t + 6755399441055744.0;  // 1.5 2^52
  const int n = (int)(uint32_t)__double_as_longlong(r);
  const double f = (r - 6755399441055744.0) - t;
  double p = x.k[10];
#pragma unroll
  for (int i = 9; i >= 0; --i) p = fma(p, f, x.k[i]);
  p = __hiloint2double(__double2hiint(p) + ((S - n) << 20), __double2loint(p));  // stays normal: n <= 900
  return (u64)__double_as_longlong(p + 4503599627370496.0) - 0x4330000000000000ull;
}
// f32 -> f64 by the bits; 0 and the subnormals become up to 2^-126, which
// changes no difference of logits.
__device__ __forceinline__ double wide(float z) {
  const uint32_t u = __float_as_uint(z);
  return __hiloint2double((int)(((u & 0x7fffffffu) >> 3) + (896u << 20) | (u & 0x80000000u)), (int)(u << 29));
}

__device__ __forceinline__ uint32_t key_of(float z) {
  const uint32_t b = __float_as_uint(z);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float z_of_key(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
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

constexpr int kPairs = 256;   // entries that are ordered by counting; one a thread
constexpr int kSegs = 1024;  // segments of a row whose kept sums are held

template <int NT>
struct SampleLds {
  union {
    struct {
      uint32_t cnt[kBins];
      u64 mass[kBins];
    };
    u64 seg[kSegs];
  };
  u64 list[kList];
  u64 wred[NT / 64 + 1], wred2[NT / 64 + 1];  // (reached_by: two words a wave)
  u64 b64[4];
  int bi[4];
};

template <int EK, int NT>
struct SampleRow {
  static constexpr int NW = NT / 64;

  const SampleArgs& a;
  SampleLds<NT>& s;
  int row;
  const uint8_t* z;  // the row's classes from `base` on, len of them
  int base, len;
  int nvec;          // vectors of 8 a thread
  float zmax;
  double zmax_w;
  double c2;         // log2(e) / T
  float inv_tf, u;
  Exp2Series series;
  // what is kept: logits above z_t, and at z_t the classes up to c_t
  float z_t = -INFINITY;
  int c_t = -1;

  __device__ __forceinline__ SampleRow(const SampleArgs& a_, SampleLds<NT>& s_, int row_, int c0, int c1)
      : a(a_), s(s_), row(row_), base(c0), len(c1 - c0) {
    z = static_cast<const uint8_t*>(a.z) + ((int64_t)row * a.ldz + c0) * (EK == EL_F32 ? 4 : 2);
    nvec = (len + NT * 8 - 1) / (NT * 8);
  }

  // The thread's vector k: classes base + (k NT + t) 8 .. +7; past the end: -inf.
  __device__ __forceinline__ int first(int k) const { return (k * NT + (int)threadIdx.x) * 8; }
  __device__ __forceinline__ int cls(int k) const { return base + first(k); }
  struct Raw {
    u32x4_t w[EK == EL_F32 ? 2 : 1];
  };
  __device__ __forceinline__ void fetch(Raw& x, int k) const {
    constexpr int ES = EK == EL_F32 ? 4 : 2;
    const int c = first(k), n = len - c;
    if (n >= 8) {
      const uint8_t* p = z + (uint32_t)c * (uint32_t)ES;
#pragma unroll
      for (int i = 0; i < (EK == EL_F32 ? 2 : 1); ++i) x.w[i] = *reinterpret_cast<const u32x4_a2*>(p + i * 16);
    } else if constexpr (EK == EL_F32) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        x.w[e >> 2][e & 3] = e < n ? reinterpret_cast<const uint32_t*>(z)[c + e] : 0xff800000u;
    } else {
      constexpr uint32_t NONE = EK == EL_F16 ? 0xfc00u : 0xff80u;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t lo = 2 * e < n ? reinterpret_cast<const uint16_t*>(z)[c + 2 * e] : NONE;
        const uint32_t hi = 2 * e + 1 < n ? reinterpret_cast<const uint16_t*>(z)[c + 2 * e + 1] : NONE;
        x.w[0][e] = lo | hi << 16;
      }
    }
  }
  __device__ __forceinline__ static float at(const Raw& x, int e) {
    if constexpr (EK == EL_F32) return __uint_as_float(x.w[e >> 2][e & 3]);
    const uint16_t h = (uint16_t)(x.w[0][(e & 7) >> 1] >> (16 * (e & 1)));
    return EK == EL_F16 ? f16_to_f32(h) : bf16_to_f32(h);
  }
  // f(k, v) for every vector of the thread, v as they are stored (the maximum
  // and comparisons leave NaN out); the next vector is on its way meanwhile.
  template <typename F>
  __device__ __forceinline__ void each_vec(F f) const {
    Raw x;
    fetch(x, 0);
#pragma unroll 1
    for (int k = 0; k < nvec; ++k) {
      Raw y = x;
      if (k + 1 < nvec) fetch(y, k + 1);
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = at(x, e);
      f(k, v);
      x = y;
    }
  }
  // f(v, class) for every element that may be drawn and is no worse than v0, until enough().
  template <typename F, typename G>
  __device__ __forceinline__ void each_from(float v0, F f, G enough) const {
    each_vec([&](int k, const float (&v)[8]) {
      float m = -INFINITY;
#pragma unroll
      for (int e = 0; e < 8; ++e) m = fmaxf(m, v[e]);
      if (!__any(m >= v0 && m > -INFINITY) || enough()) return;
#pragma unroll
      for (int e = 0; e < 8; ++e)
      {
        if (v[e] >= v0 && v[e] > -INFINITY) f(v[e], cls(k) + e);
        __builtin_amdgcn_sched_barrier(0);  // one element's work at a time: 64-bit weights take many registers
      }
    });
  }

  template <typename F>
  __device__ __forceinline__ void each_from(float v0, F f) const {
    each_from(v0, f, [] { return false; });
  }

  __device__ __forceinline__ u64 weight(float v) const {
    const u64 w = weight_of(series, (zmax_w - wide(v)) * c2, a.shift);
    return v == zmax ? 1ull << a.shift : w;
  }
  __device__ __forceinline__ static u64 comp(float v, int c) { return ((u64)(~key_of(v + 0.0f)) << 32) | (uint32_t)c; }
  __device__ __forceinline__ bool kept(float v, int c) const { return v > z_t || (v == z_t && c <= c_t); }
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

  // Fills list with the composites of the elements from v0 on that f accepts; how
  // many those are, or more than most <= kList (and the rest is not looked at).
  template <typename F>
  __device__ __forceinline__ int compact(float v0, F f, int most = kList) {
    __syncthreads();
    if (threadIdx.x == 0) s.bi[3] = 0;
    __syncthreads();
    each_from(v0, [&](float v, int c) {
      if (f(v, c)) {
        const int at = atomicAdd(&s.bi[3], 1);
        if (at < kList) s.list[at] = comp(v, c);
      }
    }, [&] { return *const_cast<volatile int*>(&s.bi[3]) > most; });
    __syncthreads();
    return s.bi[3];
  }

  // Histogram of what is kept over bin_of: the counts or the masses.
  __device__ __forceinline__ void histogram(bool by_mass) {
    clear_hist(kBins);
    if (!by_mass) {
      each_from(z_t, [&](float v, int c) {
        if (kept(v, c)) atomicAdd(&s.cnt[bin_of(v)], 1u);
      });
      return;
    }
    each_vec([&](int k, const float (&v)[8]) {
      float m = -INFINITY;
#pragma unroll
      for (int e = 0; e < 8; ++e) m = fmaxf(m, v[e]);
      if (!__any(m >= z_t && m > -INFINITY)) return;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const u64 w = weight(v[e]);
        if (kept(v[e], cls(k) + e)) {
          atomicAdd(&s.mass[bin_of(v[e])], w);
        }
        if (e & 1) __builtin_amdgcn_sched_barrier(0);
      }
    });
  }

  // Of what is kept, the target-th element (by count), or the last one before
  // which the masses add up to less than target, becomes the last one kept;
  // `cut` is the bin of bin_of that holds it.
  __device__ __forceinline__ void refine(bool by_mass, u64 target, Cut cut) {
    u64 cnt_before = cut.cnt_before, mass_before = cut.mass_before;
    int m = compact(z_t, [&](float v, int c) { return bin_of(v) == cut.bin && kept(v, c); });
    if (m > kList) {
      // the bin's members span composites [lo, hi]: 1024 bins over those, until one holds little
      u64 lo = ~0ull, hi_inv = ~0ull;
      each_from(z_t, [&](float v, int c) {
        const u64 q = comp(v, c);
        if (bin_of(v) == cut.bin && kept(v, c)) {
          lo = q < lo ? q : lo;
          hi_inv = ~q < hi_inv ? ~q : hi_inv;
        }
      });
      lo = block_min64(lo);
      u64 hi = ~block_min64(hi_inv), n = m;
      while (n > kList) {
        int shift = 64 - __clzll((long long)(hi - lo)) - 10;
        shift = shift < 0 ? 0 : shift;
        clear_hist(1024);
        each_from(z_t, [&](float v, int c) {
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
        lo += (u64)k.bin << shift;
        const u64 top = lo + ((1ull << shift) - 1);
        hi = top < hi ? top : hi;
      }
      m = compact(z_t, [&](float v, int c) {
        const u64 q = comp(v, c);
        return q >= lo && q <= hi;
      });
    }
    // of the list, what spans [lo, hi]: 1024 bins over those, until one holds few
    u64 lo = ~0ull, hi_inv = ~0ull;
    for (int i = threadIdx.x; i < m; i += NT) {
      const u64 q = s.list[i];
      lo = q < lo ? q : lo;
      hi_inv = ~q < hi_inv ? ~q : hi_inv;
    }
    lo = block_min64(lo);
    u64 hi = ~block_min64(hi_inv);
    for (int n = m; n > kPairs;) {
      int shift = 64 - __clzll((long long)(hi - lo)) - 10;
      shift = shift < 0 ? 0 : shift;
      clear_hist(1024);
      for (int i = threadIdx.x; i < m; i += NT) {
        const u64 q = s.list[i];
        if (q < lo || q > hi) continue;
        const int b = (int)((q - lo) >> shift);
        atomicAdd(&s.cnt[b], 1u);
        if (by_mass) atomicAdd(&s.mass[b], weight(z_of_key(~(uint32_t)(q >> 32))));
      }
      const Cut k = find_bin(1024, by_mass, target - (by_mass ? mass_before : cnt_before));
      cnt_before += k.cnt_before;
      mass_before += k.mass_before;
      n = k.n;
      lo += (u64)k.bin << shift;
      const u64 top = lo + ((1ull << shift) - 1);
      hi = top < hi ? top : hi;
    }
    // those few, ordered by counting
    __syncthreads();
    u64* const few = s.seg;
    u64* const w1 = s.seg + kPairs;
    if (threadIdx.x == 0) s.bi[3] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < m; i += NT) {
      const u64 q = s.list[i];
      if (q < lo || q > hi) continue;
      const int at = atomicAdd(&s.bi[3], 1);
      few[at] = q;
      w1[at] = by_mass ? weight(z_of_key(~(uint32_t)(q >> 32))) : 0;
    }
    __syncthreads();
    const int n = s.bi[3], t = threadIdx.x, some = (t & ~63) < n ? n : 0;
    const u64 q = t < n ? few[t] : ~0ull;
    u64 run = mass_before;
    int rank = 0;
#pragma unroll 4
    for (int j = 0; j < some; ++j) {
      const bool before = few[j] < q;
      rank += before;
      run += before ? w1[j] : 0;
    }
    if (t < n && (by_mass ? run < target && (run + w1[t] >= target || rank == n - 1)
                          : rank == (int)min((int64_t)(target - cnt_before), (int64_t)n) - 1))
      s.b64[2] = q;
    __syncthreads();
    z_t = z_of_key(~(uint32_t)(s.b64[2] >> 32));
    c_t = (int)(uint32_t)s.b64[2];
    __syncthreads();
  }

  __device__ __forceinline__ void write(int token, float lp) const {
    if (threadIdx.x == 0) {
      a.token[row] = token;
      if (a.logprob) a.logprob[row] = lp;
    }
  }
  __device__ __forceinline__ float log_of(float v, u64 total) const {
    const double d = v == zmax ? 0.0 : ((double)zmax - (double)v) * c2 * 0.6931471805599453;
    return (float)(-d - log(ldexp((double)total, -a.shift)));
  }
  __device__ __forceinline__ u64 draw_at(u64 total) const {
    return (u64)((double)u * (double)total);  // the sum has to pass this
  }

  // The draw where everything kept is in list[0 .. m), sorted by composite.
  __device__ __forceinline__ void draw_small(int m) {
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
        a.token[row] = (int)(q >> 32);
        if (a.logprob) a.logprob[row] = log_of(z_of_key(~(uint32_t)q), total);
      }
      run += w[i];
    }
  }

  __device__ __forceinline__ u64 kept_weight(float v, int c, u64 least) const {
    const u64 w = weight(v);
    return kept(v, c) && w >= least ? w : 0;
  }

  // The sums of what is kept with weight >= least, by segments: the classes of
  // `per` vectors of a wave, 512 each.  Segment (k / per) NW + wave.
  __device__ __forceinline__ void segment_sums(u64 least, int per) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    __syncthreads();
    u64 sum = 0;
    each_vec([&](int k, const float (&v)[8]) {
      float m = -INFINITY;
#pragma unroll
      for (int e = 0; e < 8; ++e) m = fmaxf(m, v[e]);
      if (__any(m >= z_t)) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          sum += kept_weight(v[e], cls(k) + e, least);
          if (e & 1) __builtin_amdgcn_sched_barrier(0);
        }
      }
      if ((k + 1) % per == 0 || k + 1 == nvec) {
        const u64 w = wave_sum64(sum);
        if (lane == 0) s.seg[k / per * NW + wave] = w;
        sum = 0;
      }
    });
    __syncthreads();
  }

  // The draw where seg[0 .. nseg) holds those sums of the whole row: the
  // segment that the target falls into is gone through again.  With per > 1 the
  // waves' vectors of a stretch of `per` alternate, so the stretch is.
  __device__ __forceinline__ void draw_segments(u64 least, int per, int nseg) {
    const int t = threadIdx.x, wave = t >> 6, lane = t & 63;
    auto own = [&](float v, int c) { return kept_weight(v, c, least); };
    constexpr int PER = kSegs / NT;
    u64 mine[PER], w = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      mine[i] = t * PER + i < nseg ? s.seg[t * PER + i] : 0;
      w += mine[i];
    }
    u64 run = wave_scan64(w) - w, total = 0;
    if (lane == 63) s.wred[wave] = run + w;
    if (t == 0) s.bi[0] = 0;
    __syncthreads();
    for (int k = 0; k < NW; ++k) {
      if (k < wave) run += s.wred[k];
      total += s.wred[k];
    }
    const u64 target = draw_at(total);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (run <= target && target < run + mine[i]) {
        s.bi[0] = t * PER + i;
        s.b64[0] = run;
      }
      run += mine[i];
    }
    __syncthreads();
    const int seg = s.bi[0];
    u64 before = s.b64[0];
    if (per == 1) {
      if (wave != seg % NW) return;
      Raw x;
      fetch(x, seg / NW);
      pick(x, seg / NW, before, target, total, own);
      return;
    }
    for (int q = seg / NW * NW; q < seg; ++q) before -= s.seg[q];  // the stretch's start
    for (int k = seg / NW * per; k < (seg / NW + 1) * per && k < nvec; ++k) {
      Raw x;
      fetch(x, k);
      u64 sum = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += own(at(x, e), cls(k) + e);
      sum = wave_sum64(sum);
      __syncthreads();
      if (lane == 0) s.wred[wave] = sum;
      __syncthreads();
      u64 at_wave = before;
      for (int q = 0; q < NW; ++q) {
        if (q < wave) at_wave += s.wred[q];
        before += s.wred[q];
      }
      pick(x, k, at_wave, target, total, own);
      if (before > target) return;
    }
  }

  // The draw over the row, of what is kept with weight >= least.
  __device__ __forceinline__ void draw_row(u64 least) {
    const int per = (nvec * NW + kSegs - 1) / kSegs;  // vectors a segment
    segment_sums(least, per);
    draw_segments(least, per, (nvec + per - 1) / per * NW);
  }

  // Writes the class of the wave's vector k at which the sum passes target, if
  // it is there; `run` is the sum before the wave's first.
  template <typename F>
  __device__ __forceinline__ void pick(const Raw& x, int k, u64 run, u64 target, u64 total, F own) {
    u64 w[8], sum = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      w[e] = own(at(x, e), cls(k) + e);
      sum += w[e];
    }
    run += wave_scan64(sum) - sum;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (run <= target && target < run + w[e]) {
        a.token[row] = cls(k) + e;
        if (a.logprob) a.logprob[row] = log_of(at(x, e), total);
      }
      run += w[e];
    }
  }

  // The same as finish_list for m <= kPairs (the list not sorted): an entry's place
  // in either order, and the sum before it, are counted over all entries, which
  // the lanes of a wave read from LDS together (the last launch of 1 x 131072, k 50:
  // 10.8 us; with two sorts 11.9).
  __device__ __forceinline__ void finish_pairs(int m, bool by_k, int top_k, bool by_p, float top_p, u64 mass_target,
                                               u64 least) {
    const int t = threadIdx.x, some = (t & ~63) < m ? m : 0;  // none for a wave without entries
    u64* const w1 = s.list + kPairs;
    u64* const w2 = w1 + kPairs;
    const u64 q = t < m ? s.list[t] : ~0ull;
    const u64 w = t < m ? weight(z_of_key(~(uint32_t)(q >> 32))) : 0;
    if (t < m) w1[t] = w;
    __syncthreads();
    u64 run = 0;
    int rank = 0;
#pragma unroll 4
    for (int j = 0; j < some; ++j) {
      const bool before = s.list[j] < q;
      rank += before;
      run += before ? w1[j] : 0;
    }
    const bool in = t < m && (!by_k || rank < top_k);
    u64 target = ~0ull;
    if (by_p) target = mass_target ? mass_target : (u64)ceil((double)top_p * (double)block_sum64(in ? w : 0));
    const bool keep = in && (rank == 0 || (run < target && w >= least));
    const u64 own = keep ? w : 0;
    if (t < m) w2[t] = own;
    const u64 total = block_sum64(own);
    run = 0;
#pragma unroll 4
    for (int j = 0; j < some; ++j) run += (uint32_t)s.list[j] < (uint32_t)q ? w2[j] : 0;
    const u64 at = draw_at(total);
    if (run <= at && at < run + own) {
      a.token[row] = (int)(uint32_t)q;
      if (a.logprob) a.logprob[row] = log_of(z_of_key(~(uint32_t)(q >> 32)), total);
    }
  }

  // The sorted list[0 .. m) holds all that may be kept: its last cuts and the draw.
  __device__ __forceinline__ void finish_list(int m, bool by_k, int top_k, bool by_p, float top_p, u64 least) {
    if (by_k) m = top_k < m ? top_k : m;
    if (by_p) {
      constexpr int PER = kList / NT;
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
    if (least) {  // the weights fall along the order
      int n = 0;
      for (int j = threadIdx.x; j < m; j += NT)
        if (weight(z_of_key(~(uint32_t)(s.list[j] >> 32))) >= least) ++n;
      m = (int)block_sum64((u64)n);
    }
    __syncthreads();
    draw_small(m);
  }

  // A logit that at least n elements reach, and not many more lanes' maxima than
  // n do: bisected on the keys.  1 <= n <= NT; -inf where fewer lanes have one.
  __device__ __forceinline__ float reached_by(int n, float lane_max) {
    const uint32_t key = key_of(lane_max + 0.0f);
    uint32_t* cnt = reinterpret_cast<uint32_t*>(s.wred);  // two sets of NW, in turn
    // reached by n or more (by all NT); by fewer
    uint32_t lo = key_of(-block_maxf(-lane_max) + 0.0f), hi = key_of(zmax + 0.0f) + 1;
    for (int i = 0; hi - lo > 1; ++i) {
      const uint32_t mid = lo + (hi - lo) / 2;
      const uint32_t c = (uint32_t)__popcll(__ballot(key >= mid));
      uint32_t* set = cnt + (i & 1) * NW;
      if ((threadIdx.x & 63) == 0) set[threadIdx.x >> 6] = c;
      __syncthreads();
      uint32_t all = 0;
#pragma unroll
      for (int k = 0; k < NW; ++k) all += set[k];
      if (all >= (uint32_t)n) {
        lo = mid;
        if (all <= (uint32_t)(n + n / 16)) break;
      } else {
        hi = mid;
      }
    }
    __syncthreads();
    return z_of_key(lo);
  }

  // The row's settings.
  struct Set {
    float T, top_p, min_p, u;
    int top_k;
    bool greedy, by_k, by_p;
    u64 least;
  };
  __device__ __forceinline__ static Set settings(const SampleArgs& a, int row) {
    Set q;
    q.T = a.temperature[row];
    q.u = a.u[row];
    q.top_p = a.top_p[row];
    q.min_p = a.min_p[row];
    q.top_k = a.top_k[row];
    q.greedy = !(q.T > 0.0f) || q.top_k == 1 || q.top_p <= 0.0f;
    q.by_k = q.top_k > 0 && q.top_k < a.V;
    q.by_p = q.top_p < 1.0f;
    // w >= min_p: on the rounded weights, the least whole number that min_p admits
    q.least = q.min_p > 0.0f ? (u64)ceil(ldexp((double)fminf(q.min_p, 1.0f), a.shift)) : 0;
    return q;
  }
  __device__ __forceinline__ float lane_max() {
    float m = -INFINITY;
    each_vec([&](int, const float (&v)[8]) {
#pragma unroll
      for (int e = 0; e < 8; ++e) m = fmaxf(m, v[e]);
    });
    return m;
  }
  __device__ __forceinline__ float block_maxf(float v) {
    v = wave_max(v);
    float* red = reinterpret_cast<float*>(s.wred);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int k = 1; k < NW; ++k) v = fmaxf(v, red[k]);
    __syncthreads();
    return v;
  }
  __device__ __forceinline__ int first_of_max() {
    u64 best = ~0ull;
    each_from(zmax, [&](float, int c) { best = (u64)c < best ? (u64)c : best; });
    return (int)block_min64(best);
  }
  __device__ __forceinline__ void scale_by(float zm, const Set& q) {
    zmax = zm;
    u = q.u > 0.0f ? fminf(q.u, 0.99999994f) : 0.0f;
    const double inv_t = 1.0 / (double)q.T;
    c2 = 1.4426950408889634 * inv_t;
    zmax_w = fabsf(zmax) < INFINITY ? wide(zmax) : (double)zmax;
    inv_tf = (float)inv_t;
  }
  // The draw from the list's m members, not sorted yet, which hold the top k.
  __device__ __forceinline__ void finish_top_k(int m, const Set& q) {
    if (m <= kPairs) return finish_pairs(m, true, q.top_k, q.by_p, q.top_p, 0, q.least);
    sort_list(m);
    finish_list(m, true, q.top_k, q.by_p, q.top_p, q.least);
  }
  __device__ __forceinline__ u64 mass_target(float top_p) {
    u64 own = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += NT) own += s.mass[i];
    return (u64)ceil((double)top_p * (double)block_sum64(own));
  }

  // The whole row in this workgroup; `made`: the masses' histogram is there.
  __device__ __forceinline__ void cut_and_draw(const Set& q, bool made) {
    for (int pass = 0; pass < 2; ++pass) {
      const bool by_mass = pass == 1;
      if (!(by_mass ? q.by_p : q.by_k)) continue;
      if (!made) histogram(by_mass);
      const u64 target = by_mass ? mass_target(q.top_p) : (u64)q.top_k;
      const Cut cut = find_bin(kBins, by_mass, target);
      // what lies up to the cut, if that is little
      const int most = by_mass ? kPairs : kList;
      if (by_mass || cut.cnt_before + cut.n <= kList) {
        const int m = compact(z_t, [&](float v, int c) { return bin_of(v) <= cut.bin && kept(v, c); }, most);
        if (m <= most)
          return by_mass ? finish_pairs(m, false, 0, true, q.top_p, target, q.least) : finish_top_k(m, q);
      }
      refine(by_mass, target, cut);
    }
    draw_row(q.least);
  }

  __device__ __forceinline__ void run() {
    const Set q = settings(a, row);
    const float own_max = lane_max();
    zmax = block_maxf(own_max);
    if (zmax == -INFINITY) return write(-1, -INFINITY);
    if (q.greedy) return write(first_of_max(), 0.0f);
    scale_by(zmax, q);
    if (q.by_k && q.top_k <= NT) {
      // the k largest are among what reaches a logit that k lanes' maxima reach
      const float t = reached_by(q.top_k, own_max);
      const int m = compact(t, [](float, int) { return true; });
      if (m <= kList) return finish_top_k(m, q);
    }
    cut_and_draw(q, false);
  }
};

template <int EK, int NT>
__global__ __launch_bounds__(NT) void sample_kernel(SampleArgs a) {
  __shared__ SampleLds<NT> lds;
  SampleRow<EK, NT> row(a, lds, blockIdx.x, 0, a.V);
  row.run();
}

// ---------------------------------------------------------------------------
// Few rows: P workgroups a row, in three launches.
//   1  each takes the maxima of its 16 groups of 16 lanes, and the first class
//      that has the largest; clears the row's counters
//   2  top-k: the classes that reach a logit which k of those maxima reach, into
//      the row's list; top-p alone: the row's histogram; neither: the segments'
//      sums
//   3  one workgroup a row: what is left of the cuts, and the draw (a list that
//      overflowed, or a nucleus of many classes, as without scratch)
// Scratch, in words: 0 the list's count; 16 + 20 q the q-th workgroup's (0: the
// first class of its maximum, 4 ..: the groups' maxima); 2048 the list, the
// histogram's masses, or the segments' sums.
// ---------------------------------------------------------------------------
constexpr int kPartNT = 256, kPartWords = 20, kPartAt = 16, kDataAt = 2048;
static_assert(kPartAt + 64 * kPartWords <= kDataAt, "scratch");
static_assert(kDataAt + kBins * 2 <= 8192 && kDataAt + kList * 2 <= 8192 && kDataAt + kSegs * 2 <= 8192, "scratch");

// Classes of a part: whole segments of 512.  Of ceil(V / part_len(V, P)) parts,
// only the last may have fewer.
__host__ __device__ inline int part_len(int V, int P) { return ((V + P - 1) / P + 511) & ~511; }
__device__ __forceinline__ void part_classes(int V, int P, int q, int* c0, int* c1) {
  const int len = part_len(V, P);
  *c0 = q * len;
  *c1 = min(*c0 + len, V);
}
template <int EK>
__global__ __launch_bounds__(kPartNT) void sample_part_max_kernel(SampleArgs a, uint32_t* scratch, int64_t lds, int P) {
  __shared__ SampleLds<kPartNT> sl;
  typedef SampleRow<EK, kPartNT> Row;
  const int r = blockIdx.y, q = blockIdx.x;
  int c0, c1;
  part_classes(a.V, P, q, &c0, &c1);
  Row part(a, sl, r, c0, c1);
  const typename Row::Set set = Row::settings(a, r);
  uint32_t* row = scratch + (int64_t)r * lds;
  if (q == 0 && threadIdx.x == 0) row[0] = 0;
  if (set.by_p && !set.by_k)
    for (int i = q * kPartNT + threadIdx.x; i < kBins * 2; i += P * kPartNT) row[kDataAt + i] = 0;
  const float own = part.lane_max();
  uint32_t* out = row + kPartAt + q * kPartWords;
  float w = own;
#pragma unroll
  for (int off = 8; off > 0; off >>= 1) w = fmaxf(w, __shfl_xor(w, off, 64));
  if ((threadIdx.x & 15) == 0) out[4 + (threadIdx.x >> 4)] = __float_as_uint(w);
  if (set.greedy) {
    part.zmax = part.block_maxf(own);
    const int at = part.zmax > -INFINITY ? part.first_of_max() : -1;
    if (threadIdx.x == 0) out[0] = (uint32_t)at;
  }
}

// The groups' maxima of a row's parts, those of part `lane` in each lane.
constexpr int kGroups = 16;
__device__ __forceinline__ void parts_max(const uint32_t* row, int P, float (&m)[kGroups]) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int i = 0; i < kGroups; i += 4) {
    f32x4 v = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    if (lane < P) v = *reinterpret_cast<const f32x4_a4*>(row + kPartAt + lane * kPartWords + 4 + i);
#pragma unroll
    for (int e = 0; e < 4; ++e) m[i + e] = v[e];
  }
}
__device__ __forceinline__ float max_of(const float (&m)[kGroups]) {
  float t = m[0];
#pragma unroll
  for (int i = 1; i < kGroups; ++i) t = fmaxf(t, m[i]);
  return t;
}
// A logit that n of them reach (n <= 16 P; -inf where fewer are there), and not
// many more: bisected on the keys, in each wave for itself.
__device__ __forceinline__ float reached_by_parts(const float (&m)[kGroups], int P, float zmax, int n) {
  uint32_t key[kGroups];
#pragma unroll
  for (int i = 0; i < kGroups; ++i) key[i] = key_of(m[i] + 0.0f);
  // reached by all 16 P, or by n; by fewer
  float low = INFINITY;
#pragma unroll
  for (int i = 0; i < kGroups; ++i) low = fminf(low, m[i]);
  low = -wave_max((int)(threadIdx.x & 63) < P ? -low : -INFINITY);
  uint32_t lo = key_of(low + 0.0f), hi = key_of(zmax + 0.0f) + 1;
  while (hi - lo > 1) {
    const uint32_t mid = lo + (hi - lo) / 2;
    int c = 0;
#pragma unroll
    for (int i = 0; i < kGroups; ++i) c += __popcll(__ballot(key[i] >= mid));
    if (c >= n) {
      lo = mid;
      if (c <= n + n / 16) break;
    } else {
      hi = mid;
    }
  }
  return z_of_key(lo);
}

template <int EK>
__global__ __launch_bounds__(kPartNT) void sample_part_kernel(SampleArgs a, uint32_t* scratch, int64_t lds, int P) {
  __shared__ SampleLds<kPartNT> sl;
  typedef SampleRow<EK, kPartNT> Row;
  const int r = blockIdx.y, q = blockIdx.x;
  const typename Row::Set set = Row::settings(a, r);
  uint32_t* row = scratch + (int64_t)r * lds;
  float maxima[kGroups];
  parts_max(row, P, maxima);
  const float zmax = wave_max(max_of(maxima));
  if (set.greedy || zmax == -INFINITY) return;
  int c0, c1;
  part_classes(a.V, P, q, &c0, &c1);
  Row part(a, sl, r, c0, c1);
  part.scale_by(zmax, set);
  u64* data = reinterpret_cast<u64*>(row + kDataAt);
  if (set.by_k) {
    if (set.top_k > kGroups / 2 * P) return;  // the third launch takes it whole
    const float t = reached_by_parts(maxima, P, zmax, set.top_k);
    const int m = part.compact(t, [](float, int) { return true; });
    if (threadIdx.x == 0) sl.bi[0] = m > 0 ? (int)atomicAdd(row, (uint32_t)m) : 0;
    __syncthreads();
    const int at = sl.bi[0], n = min(m, kList);
    for (int i = threadIdx.x; i < n && at + i < kList; i += kPartNT) data[at + i] = sl.list[i];
  } else if (set.by_p) {
    part.histogram(true);
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += kPartNT)
      if (sl.mass[i]) atomicAdd(data + i, sl.mass[i]);
  } else {
    part.segment_sums(set.least, 1);
    const int nseg = (c1 - c0 + 511) / 512;
    for (int i = threadIdx.x; i < nseg; i += kPartNT) data[c0 / 512 + i] = sl.seg[i];
  }
}

template <int EK>
__global__ __launch_bounds__(1024) void sample_join_kernel(SampleArgs a, const uint32_t* scratch, int64_t lds, int P) {
  constexpr int NT = 1024;
  __shared__ SampleLds<NT> sl;
  typedef SampleRow<EK, NT> Row;
  const int r = blockIdx.x, lane = threadIdx.x & 63;
  const uint32_t* row = scratch + (int64_t)r * lds;
  Row whole(a, sl, r, 0, a.V);
  const typename Row::Set set = Row::settings(a, r);
  // on their way with the settings, before it is known that there is a list
  const u64* data = reinterpret_cast<const u64*>(row + kDataAt);
  const uint32_t m = row[0];
  const u64 entry = data[threadIdx.x];
  float maxima[kGroups];
  parts_max(row, P, maxima);
  const float part_max = max_of(maxima), zmax = wave_max(part_max);
  if (zmax == -INFINITY) return whole.write(-1, -INFINITY);
  if (set.greedy) {
    uint32_t at = lane < P && part_max == zmax ? row[kPartAt + lane * kPartWords] : 0xffffffffu;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) at = min(at, (uint32_t)__shfl_xor((int)at, off, 64));
    return whole.write((int)at, 0.0f);
  }
  whole.scale_by(zmax, set);
  if (set.by_k) {
    if (set.top_k > kGroups / 2 * P || m > kList) return whole.run();
    if (threadIdx.x < m) sl.list[threadIdx.x] = entry;
    if (threadIdx.x + NT < m) sl.list[threadIdx.x + NT] = data[threadIdx.x + NT];
    __syncthreads();
    return whole.finish_top_k((int)m, set);
  }
  if (set.by_p) {
    for (int i = threadIdx.x; i < kBins; i += NT) sl.mass[i] = data[i];
    __syncthreads();
    return whole.cut_and_draw(set, true);
  }
  const int nseg = (a.V + 511) / 512;
  for (int i = threadIdx.x; i < nseg; i += NT) sl.seg[i] = data[i];
  __syncthreads();
  whole.draw_segments(set.least, 1, nseg);
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
Status sample_run(const SampleArgs& a, uint32_t* scratch, int64_t lds, hipStream_t s) {
  const unsigned g = (unsigned)a.R;
  // Few long rows share the chip: parts of 2048 classes or more, about one
  // workgroup a CU.  A row a workgroup against this, bf16: plain draws 1 x 40000
  // 23.9 us (15.2), 1 x 262144 93.1 (15.2), 32 x 65536 32.2 (17.8); top-p 0.9 1 x
  // 262144 257.6 (180.5), 32 x 65536 87.5 (78.4); top-k 50 32 x 131072 27.3 (25.5),
  // 1 x 40000 17.6 (23.3), 64 x 131072 27.8 (42.2).  The settings are on the
  // device; below 32768 classes and beyond 32 rows top-k loses more than others
  // gain.
  int P = 256 / a.R;
  if (P > a.V / 2048) P = a.V / 2048;
  if (P > 64) P = 64;
  if (scratch && a.R <= 32 && a.V >= 32768 && a.V <= 512 * kSegs) {
    P = (a.V + part_len(a.V, P) - 1) / part_len(a.V, P);
    const dim3 grid((unsigned)P, g);
    sample_part_max_kernel<EK><<<grid, kPartNT, 0, s>>>(a, scratch, lds, P);
    sample_part_kernel<EK><<<grid, kPartNT, 0, s>>>(a, scratch, lds, P);
    sample_join_kernel<EK><<<g, 1024, 0, s>>>(a, scratch, lds, P);
    return launch_status("sample_row");
  }
  // Short rows, and several rows a CU: 256 threads; else 1024.  256 against 1024,
  // bf16, plain draws and top-p 0.9: 64 x 2000 7.7 us (15.3), 10.8 (19.2); 64 x
  // 16384 16.1 (17.2), 33.4 (31.1); 2048 x 50021 161.5 (268.2), 325.7 (437.7); the
  // other way 256 x 32000 28.3 (26.8), 83.6 (59.3).  At 512 x 131072 126.3 (124.1),
  // 346.3 (313.5), top-k 50 61.5 (66.5).
  if (a.V <= 16384 || a.R >= 512) sample_kernel<EK, 256><<<g, 256, 0, s>>>(a);
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
  uint32_t* scratch = no > 2 && aligned(out[2].data, 8) && out[2].shape[1] % 2 == 0 ? (uint32_t*)out[2].data : nullptr;
  const int64_t lds = no > 2 ? out[2].shape[1] : 0;
  if (ek == EL_F32) return sample_run<EL_F32>(a, scratch, lds, s);
  return ek == EL_F16 ? sample_run<EL_F16>(a, scratch, lds, s) : sample_run<EL_BF16>(a, scratch, lds, s);
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
