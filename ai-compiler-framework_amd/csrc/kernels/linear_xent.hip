// Softmax cross-entropy of a vocabulary head from its hidden rows and weights,
// with the gradients of both; the logits are not kept.
//
//   z = X W^T [R, V] (f32 sums),  lse_r = log sum_v exp z_rv
//   row loss_r = lse_r - z_{r, label},  loss = sum_r w_r row loss_r
//   G = w_r (exp(z - lse) - onehot(label)),  dX = G W,  dW = G^T X
//
// The rows that count (a label, a weight other than 0) are gathered first, so
// that the others cost nothing and nothing in them reaches a product; how many
// they are only the device knows, and the products' grids cover all rows.
//
//   1. logits: tiles of the MFMA GEMM whose epilogue keeps, for each row and
//      tile of classes, the maximum and the sum of exp(z - maximum); of some
//      classes also exp(z - tile maximum) itself (f32, or f16 for operands of
//      16 bits: 2^-11 against the 2^-8 of a bf16 G; the sums are taken before
//      the rounding): of the last `piece` in scratch, of the first `held` in the
//      memory of dW's other rows, which are written later;
//   2. the row's statistics are joined; the kept values become G in place,
//      scaled by what makes the largest weight 1 (f16: 2^13), which the products
//      take out again (weights of 1/R would leave f16's range);
//   3. dW and dX of those classes;
//   4. the other pieces: logits once more, whose epilogue knows the row's
//      statistics and writes G, then dW and dX as before.
// So the memory decides what is computed twice: 6 n V D operations where it
// holds all classes (n rows that count), up to 8 n V D where it holds few.  At
// 8192 x 131072 x 4096 bf16 and 1.5 GiB scratch holds 58% of the classes and dW
// 33%: 20.7 ms; with the 42% behind scratch alone kept it took 23.0.
// dX is summed over the pieces, and over shares of the classes where its tiles
// are fewer than the CUs, in f32 slabs that are joined in a fixed order.
//
// No counterpart in the reference.
#include <algorithm>

#include "../common/gemm_nt.hpp"
#include "../common/head_util.hpp"

namespace aicf::hip {

namespace {

constexpr float kLog2e = 1.4426950408889634f;

// 2^((z - m) log2 e): the difference first, so that the exponent is off by
// roundings of itself alone however far the logits lie from zero.
__device__ __forceinline__ float exp_from(float z, float m) { return __builtin_amdgcn_exp2f((z - m) * kLog2e); }
// The exponentials kept in f16 are at most 2^14, so that they lose bits only below 2^-28 of their tile's largest.
constexpr float kKeepScale = 16384.0f;
// A maximum over nothing but -inf is no reference: their exponentials are 0.
__device__ __forceinline__ float safe_ref(float m) { return m == -INFINITY ? 0.0f : m; }
// What a sum of exp(z - m) is multiplied by where the reference becomes `to`.
__device__ __forceinline__ float rebase(float m, float to) { return m == -INFINITY ? 0.0f : exp_from(m, to); }

// ---------------------------------------------------------------------------
// The products' epilogues
// ---------------------------------------------------------------------------
template <int OUT, int ACT, int BM, int BN, int WM, int WN, int STAGE_BYTES, int MS>
__device__ __forceinline__ void lx_epilogue(const NTParams& p, nt_acc_t<MS> (&acc)[BN / WN / MS][BM / WM / MS],
                                            uint8_t* smem, int m0, int n0) {
  constexpr int NW = WM * WN, NT = 64 * NW;
  constexpr int WTM = BM / WM, WTN = BN / WN;
  constexpr int TM = WTM / MS, TN = WTN / MS;
  constexpr int G = MS == 32 ? 4 : 1;  // quads of columns a block (see nt_epilogue_staged)
  constexpr int OB = OUT == OUT_F32 ? 4 : 2;
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));  // nothing of the epilogue is computed before the K loop
  const int lane = tid & 63, wave = tid >> 6;
  const int wm = wave / WN, wn = wave % WN;
  const int fr = lane % MS, fh = lane / MS;
  auto col_of = [&](int i, int g) -> int { return wn * WTN + i * MS + (MS == 32 ? 8 * g + 4 * fh : 4 * fh); };
  auto row_of = [&](int j) -> int { return wm * WTM + j * MS + fr; };

  const int ncol = p.N - n0;  // classes (columns) of the tile
  // Accumulators are read where they are used and never written: changed in
  // place, the 256 of a lane of the four-wave tiles went through a second set.
  auto value = [&](auto TAIL, int i, int j, int r) -> float {
    if constexpr (decltype(TAIL)::value)
      return col_of(i, r >> 2) + (r & 3) < ncol ? acc[i][j][r] : -INFINITY;
    return acc[i][j][r];
  };

  if constexpr (ACT == ACT_LX_STATS) {
    float* red_m = reinterpret_cast<float*>(smem);  // [WN][BM]
    float* red_s = red_m + WN * BM;
    static_assert(2 * WN * BM * 4 <= STAGE_BYTES, "the waves' statistics fit");
    auto maxima = [&](auto TAIL) {
#pragma unroll
      for (int j = 0; j < TM; ++j) {
        float m = -INFINITY;
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
          for (int r = 0; r < 4 * G; ++r) m = fmaxf(m, value(TAIL, i, j, r));
        if constexpr (MS == 16) m = fmaxf(m, __shfl_xor(m, 16, 64));
        m = fmaxf(m, __shfl_xor(m, 32, 64));
        if (fh == 0) red_m[wn * BM + row_of(j)] = m;
      }
    };
    auto sums = [&](auto TAIL) {
#pragma unroll
      for (int j = 0; j < TM; ++j) {
        float m = red_m[row_of(j)];
#pragma unroll
        for (int w = 1; w < WN; ++w) m = fmaxf(m, red_m[w * BM + row_of(j)]);
        m = safe_ref(m);
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
          for (int r = 0; r < 4 * G; ++r) s += exp_from(value(TAIL, i, j, r), m);
        if constexpr (MS == 16) s += __shfl_xor(s, 16, 64);
        s += __shfl_xor(s, 32, 64);
        if (fh == 0) red_s[wn * BM + row_of(j)] = s;
      }
    };
    const bool tail = ncol < BN;
    if (tail) maxima(std::true_type{});
    else maxima(std::false_type{});
    // the label's logit: one lane of one tile has it
#pragma unroll
    for (int j = 0; j < TM; ++j) {
      const int m = m0 + row_of(j);
      const int c = (m < p.M ? p.lx.label[m] - p.lx.v0 - n0 : -1) - wn * WTN;
      if (c >= 0 && c < WTN && ((c >> 2) & (64 / MS - 1)) == fh) {
        float z = 0.0f;
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
          for (int r = 0; r < 4 * G; ++r)
            z = c == i * MS + (MS == 32 ? 8 * (r >> 2) : 0) + 4 * fh + (r & 3) ? acc[i][j][r] : z;
        p.lx.zlab[m] = z;
      }
    }
    __syncthreads();
    if (tail) sums(std::true_type{});
    else sums(std::false_type{});
    __syncthreads();
    for (int t = tid; t < BM; t += NT) {
      float m = red_m[t], s = red_s[t];
#pragma unroll
      for (int w = 1; w < WN; ++w) {
        m = fmaxf(m, red_m[w * BM + t]);
        s += red_s[w * BM + t];
      }
      p.lx.stats[(int64_t)((p.lx.v0 + n0) / BN) * p.lx.stats_ld + m0 + t] = make_float2(m, s);
    }
    if (n0 < p.lx.keep_from) return;
  }

  // Through LDS, so that whole rows are stored (as nt_epilogue_staged does).
  // A pass' four columns of a lane, v[4], from the row's constants c.
  struct RowConst {
    float a, f, w;  // reference or factor; G: factor and the label's value
    int col;        // G: the label's column
  };
  auto row_const = [&](int j) -> RowConst {
    RowConst c{0.0f, 0.0f, 0.0f, -1};
    const int m = m0 + row_of(j);
    if constexpr (ACT == ACT_LX_STATS) {
      const float* red_m = reinterpret_cast<const float*>(smem);
      c.a = red_m[row_of(j)];
#pragma unroll
      for (int w = 1; w < WN; ++w) c.a = fmaxf(c.a, red_m[w * BM + row_of(j)]);
      c.a = safe_ref(c.a);
    } else if constexpr (ACT == ACT_LX_GRAD) {
      if (m < p.M) {
        c.a = safe_ref(p.lx.row_max[m]);
        c.f = p.lx.row_f[m];
        c.w = p.lx.row_g[m];
        c.col = p.lx.label[m] - p.lx.v0 - n0;
      }
    } else if constexpr (ACT == ACT_LX_OUT) {
      c.a = p.lx.alpha[0];
    }
    return c;
  };
  auto result = [&](const RowConst& c, int i, int j, int g, int e) -> float {
    const float z = acc[i][j][4 * g + e];
    const int col = col_of(i, g) + e;
    if constexpr (ACT == ACT_LX_STATS) {
      const float v = exp_from(col < ncol ? z : -INFINITY, c.a);
      return OUT == OUT_F32 ? v : v * kKeepScale;
    } else if constexpr (ACT == ACT_LX_GRAD) {
      const float v = exp_from(z, c.a) * c.f;
      return col < ncol ? (col == c.col ? c.w : v) : 0.0f;
    } else if constexpr (ACT == ACT_LX_OUT) {
      return z * c.a;
    } else {
      return z;
    }
  };
  RowConst rc[TM];
#pragma unroll
  for (int j = 0; j < TM; ++j) rc[j] = row_const(j);
  if constexpr (ACT == ACT_LX_STATS) __syncthreads();  // the maxima are read: the stage is free
  constexpr int ROWB = BN * OB, CPR = ROWB / 16, CE = 16 / OB;
  constexpr int ROWS_PASS = STAGE_BYTES / ROWB < BM ? STAGE_BYTES / ROWB : BM;
  constexpr int NPASS = BM / ROWS_PASS, JP = TM / NPASS, WROWS = JP * MS;
  static_assert(NPASS * ROWS_PASS == BM && JP * NPASS == TM, "pass split");
  static_assert((CPR & (CPR - 1)) == 0 && (ROWS_PASS * CPR) % NT == 0, "chunk split");
  typedef typename std::conditional<OB == 4, float, uint16_t>::type out_t;
#pragma unroll
  for (int pass = 0; pass < NPASS; ++pass) {
#pragma unroll
    for (int jj = 0; jj < JP; ++jj)
#pragma unroll
      for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const int j = pass * JP + jj;
          float v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = result(rc[j], i, j, g, e);
          const int pr = wm * WROWS + jj * MS + fr, cb = col_of(i, g) * OB;
          uint8_t* at = smem + pr * ROWB + (((cb / 16) ^ (pr & (CPR - 1))) * 16) + cb % 16;
          if constexpr (OUT == OUT_F32) {
            *reinterpret_cast<f32x4*>(at) = f32x4{v[0], v[1], v[2], v[3]};
          } else if constexpr (OUT == OUT_BF16 && ACT != ACT_LX_STATS) {
            typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
            *reinterpret_cast<u32x2*>(at) = u32x2{f32x2_to_bf16x2(v[0], v[1]), f32x2_to_bf16x2(v[2], v[3])};
          } else {
            *reinterpret_cast<u16x4*>(at) = u16x4{f32_to_f16(v[0]), f32_to_f16(v[1]), f32_to_f16(v[2]), f32_to_f16(v[3])};
          }
        }
    __syncthreads();
#pragma unroll 4
    for (int k = 0; k < ROWS_PASS * CPR / NT; ++k) {
      const int idx = tid + k * NT, pr = idx / CPR, c = idx % CPR;
      const u16x8 x = *reinterpret_cast<const u16x8*>(smem + pr * ROWB + ((c ^ (pr & (CPR - 1))) * 16));
      const int m = m0 + (pr / WROWS) * WTM + pass * WROWS + (pr % WROWS);
      if (m >= p.M) continue;
      if constexpr (ACT == ACT_LX_SLAB) {
        const int n = n0 + c * CE;
        if (n >= p.ldc) continue;  // (a slab's rows are whole 64s)
        f32x4* q = reinterpret_cast<f32x4*>((float*)p.C + (int64_t)m * p.ldc + n);
        f32x4 v = __builtin_bit_cast(f32x4, x);
        if (p.lx.add) v += *q;
        *q = v;
      } else if constexpr (ACT != ACT_LX_OUT) {  // G's rows hold whole tiles
        out_t* q = (out_t*)p.C + (int64_t)m * p.ldc + (n0 - (ACT == ACT_LX_STATS ? p.lx.keep_from : 0)) + c * CE;
        *reinterpret_cast<u16x8*>(q) = x;
      } else {
        const int n = n0 + c * CE;
        const int64_t row = p.lx.row_map ? p.lx.row_map[m] : m;
        out_t* q = (out_t*)p.C + row * p.ldc + n;
        if (p.lx.vec && n + CE <= p.N) {
          *reinterpret_cast<u16x8*>(q) = x;
        } else {
#pragma unroll
          for (int e = 0; e < CE; ++e)
            if (n + e < p.N) {
              if constexpr (OUT == OUT_F32) q[e] = __builtin_bit_cast(f32x4, x)[e];
              else q[e] = x[e];
            }
        }
      }
    }
    if (pass + 1 < NPASS) __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// Rows
// ---------------------------------------------------------------------------
// Scratch of a call, in this order; every array starts on 256 bytes.
struct LxRows {
  int32_t* head;    // [0] rows that count; f32 [1] what the products with G are multiplied by, [2] its inverse,
                    // [3] 1 / rows that count; [4] shares of dX's K
  int32_t* idx;     // [Rp] rows that count, in their order
  int32_t* label;   // [Rp] theirs, like all below
  float* weight;    // as given
  float* row_g;     // G of the label, from its f32 logit
  float* zlab;
  float* row_max;
  float* row_f;     // weight head[2] / sum of exp(z - row_max)
  float* row_loss;
  float2* stats;    // [tiles of classes][Rp]
  void* xc;         // [Rp][Dp] rows of X, zeros behind D
  float* slab;      // dX in f32, one for each share of the classes
  void* wpad;       // [piece][Dp] rows of W, where W itself cannot be read in tiles
  void* g;          // [Rp][piece]
};

template <int ES>
struct LxElem;
template <>
struct LxElem<2> {
  typedef uint16_t T;
  typedef u16x8 vec;
  typedef u16x8_a2 loose;
};
template <>
struct LxElem<4> {
  typedef float T;
  typedef f32x4 vec;
  typedef f32x4_a4 loose;
};

struct LxCopy {
  const void* src;
  void* dst;   // [.][Dp], 16-byte steps
  void* dx;    // nullptr: none
  float* row_loss;
  int64_t lds, lddx;
  int D, Dp;
};

// 16 bytes from element i of row r of src (D elements), zeros behind them.
template <int ES>
__device__ __forceinline__ typename LxElem<ES>::vec lx_load_part(const LxCopy& c, int64_t r, int i) {
  typedef typename LxElem<ES>::T T;
  const T* a = (const T*)c.src + r * c.lds;
  if (i + 16 / ES <= c.D) return *reinterpret_cast<const typename LxElem<ES>::loose*>(a + i);
  typename LxElem<ES>::vec v;
#pragma unroll
  for (int e = 0; e < 16 / ES; ++e) v[e] = i + e < c.D ? a[i + e] : T(0);
  return v;
}

// They go to row `to` of dst; to < 0: a row that is left out, whose gradient and
// loss are cleared.
template <int ES>
__device__ __forceinline__ void lx_store_part(const LxCopy& c, int64_t r, int to, int i,
                                              const typename LxElem<ES>::vec& v) {
  typedef typename LxElem<ES>::T T;
  if (to >= 0) {
    if (i < c.Dp) *reinterpret_cast<typename LxElem<ES>::vec*>((T*)c.dst + (int64_t)to * c.Dp + i) = v;
    return;
  }
  if (i == 0) c.row_loss[r] = 0.0f;
  if (!c.dx) return;
  T* b = (T*)c.dx + r * c.lddx;
  if (i + 16 / ES <= c.D) {
    typename LxElem<ES>::loose z;
#pragma unroll
    for (int e = 0; e < 16 / ES; ++e) z[e] = T(0);
    *reinterpret_cast<typename LxElem<ES>::loose*>(b + i) = z;
  } else {
    for (int e = 0; i + e < c.D; ++e) b[i + e] = T(0);
  }
}

// Rows of W onto 16-byte steps, or (with pos) rows of X to their places.
template <int ES>
__global__ __launch_bounds__(256) void lx_copy_rows_kernel(LxCopy c, int rows, const int32_t* __restrict__ pos) {
  const int r = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r >= rows) return;
  const int to = pos ? pos[r] : r;
  for (int i = (threadIdx.x & 63) * (16 / ES); i < c.Dp; i += 64 * (16 / ES)) {
    typename LxElem<ES>::vec v{};
    if (to >= 0) v = lx_load_part<ES>(c, r, i);
    lx_store_part<ES>(c, r, to, i, v);
  }
}

// How dX's tiles are shared out: tiles of bm rows, tiles_n in a row of them,
// `slots` workgroups run at once, K (the classes of the longest part), rows that
// all slabs together may have.
struct LxShares {
  int bm, tiles_n, slots, k_piece, slab_rows;
};

// Which rows count, the factor that makes the largest weight 2^top, how many shares dX's K is divided into; and the rows of X
// to their places.  Every workgroup counts all rows (PER a thread at a time: 32
// KB of labels and weights at 4096 rows, from L2) and copies kCopyRows of them
// at most; the first one writes what the others computed too.  64 rows of 2048
// f16 take 5 us (counted and copied by one workgroup 14.5), three quarters of 4096
// rows of 4096 bf16 18 (in two launches 23 and what lies between them).
// Above kCountedByAll rows the counting, which grows with their square, is done by
// one workgroup that leaves the places in pos, and the copy by another launch
// (262144 rows of 64 bf16 522 -> 192 us; 65536 44 either way).
constexpr int kCountedByAll = 32768, kCopyRows = kCountedByAll / 256;
template <int ES, int PER>
__global__ __launch_bounds__(1024) void lx_rows_kernel(const int32_t* __restrict__ labels,
                                                       const float* __restrict__ w, int R, int V, int top, LxRows s,
                                                       LxShares sh, LxCopy cp, int per,
                                                       int32_t* __restrict__ pos) {
  __shared__ int place[kCopyRows];
  const bool first = blockIdx.x == 0;
  const int r0 = blockIdx.x * per;
  __shared__ int cnt[PER * 16 + 1];
  __shared__ float big[16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float most = 0.0f;
  int total = 0;
  for (int base = 0; base < R; base += PER * 1024) {
    int label[PER];
    uint64_t in[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int r = base + k * 1024 + threadIdx.x;
      label[k] = r < R ? labels[r] : -1;
      const float wr = r < R && w ? w[r] : 1.0f;
      const bool c = label[k] >= 0 && label[k] < V && wr != 0.0f;
      if (c) most = fmaxf(most, fabsf(wr));
      in[k] = __ballot(c);
      if (lane == 0) cnt[k * 16 + wave] = __popcll(in[k]);
    }
    __syncthreads();
    if (wave == 0) {  // places of the groups of 64 rows, in the rows' order
      int before[(PER * 16 + 63) / 64], sum = 0;
      constexpr int EACH = (PER * 16 + 63) / 64;
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
        const int at = lane * EACH + i;
        before[i] = sum;
        sum += at < PER * 16 ? cnt[at] : 0;
      }
      int up = sum;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const int o = __shfl_up(up, off, 64);
        if (lane >= off) up += o;
      }
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
        const int at = lane * EACH + i;
        if (at < PER * 16) cnt[at] = total + up - sum + before[i];
      }
      if (lane == 63) cnt[PER * 16] = total + up;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int r = base + k * 1024 + threadIdx.x;
      if (r >= R) continue;
      const bool c = in[k] >> lane & 1;
      const int at = cnt[k * 16 + wave] + __popcll(in[k] & ((1ull << lane) - 1));
      if (r >= r0 && r < r0 + per) place[r - r0] = c ? at : -1;
      if (pos) pos[r] = c ? at : -1;
      if (first && c) {
        s.idx[at] = r;
        s.label[at] = label[k];
        if (w) s.weight[at] = w[r];
      }
    }
    total = cnt[PER * 16];
    __syncthreads();
  }
  if (first) {
    most = wave_max(most);
    if (lane == 0) big[wave] = most;
    __syncthreads();
  }
  if (first && wave == 0) {
    float m = big[lane & 15];
    m = wave_max(m);
    const float mean = total > 0 ? 1.0f / (float)total : 0.0f;
    if (!w) m = mean;
    // 2^top / m, so that the largest weight (all of them, in a mean) has no
    // rounding in G, which all products with its row would share; a power of
    // two where the quotient is no normal number.
    float up = ldexpf(1.0f / m, top), down = ldexpf(m, -top);
    if (!(m > 0x1p-100f && m < 0x1p100f)) {
      int e = 0;
      if (m > 0.0f && m < INFINITY) frexpf(m, &e);  // m < 2^e
      e = top - e;
      e = e > 126 ? 126 : e < -126 ? -126 : e;
      up = ldexpf(1.0f, e);
      down = ldexpf(1.0f, -e);
    }
    // Shares: rounds of the workgroups that run at once, times a share's K-steps
    // and some 8 for a tile's first loads and its end; a share's sums are
    // written and read once more (1/32 of a step a tile when all CUs do it).
    const int tiles = (total + sh.bm - 1) / sh.bm * sh.tiles_n, k = lane + 1;
    const int steps = (sh.k_piece + 63) / 64;
    float cost = INFINITY;
    if (k == 1 || (steps / k >= 8 && (int64_t)k * ((total + sh.bm - 1) / sh.bm * sh.bm) <= sh.slab_rows &&
                   tiles * k <= 4 * sh.slots))
      cost = (float)((tiles * k + sh.slots - 1) / sh.slots) * (float)((steps + k - 1) / k + 8) +
             (k > 1 ? 4.0f + (float)(tiles * k) * (8.0f / 256.0f) : 0.0f);
    int best = k;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
      const float oc = __shfl_xor(cost, off, 64);
      const int ok = __shfl_xor(best, off, 64);
      if (oc < cost || (oc == cost && ok < best)) {
        cost = oc;
        best = ok;
      }
    }
    if (lane == 0) {
      s.head[0] = total;
      s.head[1] = __float_as_int(down);
      s.head[2] = __float_as_int(up);
      s.head[3] = __float_as_int(mean);
      s.head[4] = best;
    }
  }
  constexpr int SEG = 64 * (16 / ES);  // (place[]: behind the last chunk's barrier)
  const int segs = (cp.Dp + SEG - 1) / SEG, rows = R - r0 < per ? R - r0 : per;
  for (int t0 = wave; t0 < rows * segs; t0 += 64) {  // four loads in flight
    typename LxElem<ES>::vec v[4];
    int to[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int t = t0 + 16 * u, k = t / segs;
      to[u] = t < rows * segs ? place[k] : -1;
      if (to[u] >= 0) v[u] = lx_load_part<ES>(cp, r0 + k, (t - k * segs) * SEG + lane * (16 / ES));
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int t = t0 + 16 * u, k = t / segs;
      if (t < rows * segs) lx_store_part<ES>(cp, r0 + k, to[u], (t - k * segs) * SEG + lane * (16 / ES), v[u]);
    }
  }
}

// The statistics of a row's tiles joined: 64 rows a workgroup, wave w takes
// tiles w, w + 16, ..., eight loads in flight; the waves in order.  loss (at
// most 64 rows, one workgroup): their weighted sum too.
__global__ __launch_bounds__(1024) void lx_stats_kernel(LxRows s, int tiles, int64_t ld, bool weights,
                                                        float* __restrict__ row_loss, float* __restrict__ loss) {
  __shared__ float2 red[16][64];
  const int n = s.head[0], lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = blockIdx.x * 64 + lane;
  if (blockIdx.x * 64 >= n) {
    if (loss && threadIdx.x == 0) loss[0] = 0.0f;
    return;
  }
  float m = -INFINITY, sum = 0.0f;
  for (int t0 = wave; t0 < tiles; t0 += 16 * 8) {
    float2 v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int t = t0 + u * 16;  // (rows behind n: whatever is there, not used)
      v[u] = t < tiles ? s.stats[(int64_t)t * ld + r] : make_float2(-INFINITY, 0.0f);
    }
    float top = m;
#pragma unroll
    for (int u = 0; u < 8; ++u) top = fmaxf(top, v[u].x);
    const float ref = safe_ref(top);
    sum *= rebase(m, ref);
#pragma unroll
    for (int u = 0; u < 8; ++u) sum += v[u].y * rebase(v[u].x, ref);
    m = top;
  }
  red[wave][lane] = make_float2(m, sum);
  __syncthreads();
  if (wave > 0) return;
  float part = 0.0f, weight = 0.0f;
  if (r < n) {
    m = red[0][lane].x;
#pragma unroll
    for (int w = 1; w < 16; ++w) m = fmaxf(m, red[w][lane].x);
    const float ref = safe_ref(m);
    sum = 0.0f;
#pragma unroll
    for (int w = 0; w < 16; ++w) sum += red[w][lane].y * rebase(red[w][lane].x, ref);
    weight = weights ? s.weight[r] : __int_as_float(s.head[3]);
    const float up = weight * __int_as_float(s.head[2]);
    s.row_max[r] = m;
    s.row_f[r] = up / sum;
    s.row_g[r] = exp_from(s.zlab[r], ref) * (up / sum) - up;
    part = logf(sum) + (ref - s.zlab[r]);
    s.row_loss[r] = part;
    if (!weights) s.weight[r] = weight;
    row_loss[s.idx[r]] = part;
  }
  if (!loss) return;
  double v = (double)weight * (double)part;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  if (lane == 0) loss[0] = (float)v;
}

// loss = sum of weight * row loss, in f64 and a fixed order.
__global__ __launch_bounds__(1024) void lx_loss_kernel(LxRows s, float* __restrict__ loss) {
  __shared__ double red[16];
  const int n = s.head[0];
  double v = 0.0;
  for (int r = threadIdx.x; r < n; r += 1024) v += (double)s.weight[r] * (double)s.row_loss[r];
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  if (threadIdx.x == 0) {
    v = red[0];
    for (int i = 1; i < 16; ++i) v += red[i];
    loss[0] = (float)v;
  }
}

// The kept exp(z - tile maximum) of classes v0 .. v0 + cols become G in place.
// A lane takes 16 bytes; a tile of BN classes has one factor a row.
template <int EK, int BN>
__global__ __launch_bounds__(256) void lx_scale_kernel(LxRows s, void* g, int64_t ldg, int width, int v0,
                                                       int64_t stats_ld) {
  constexpr int ES = EK == EL_F32 ? 4 : 2, CE = 16 / ES;
  typedef typename LxElem<ES>::T T;
  typedef typename LxElem<ES>::vec vec;
  const int n = s.head[0];
  const int c = (blockIdx.x * 256 + threadIdx.x) * CE;
  if (c >= width) return;
  for (int r = blockIdx.y; r < n; r += gridDim.y) {
    const float2 st = s.stats[(int64_t)((v0 + c) / BN) * stats_ld + r];
    const float f = rebase(st.x, safe_ref(s.row_max[r])) * s.row_f[r] * (EK == EL_F32 ? 1.0f : 1.0f / kKeepScale);
    T* q = (T*)g + (int64_t)r * ldg + c;
    vec x = *reinterpret_cast<const vec*>(q);
    const int at = s.label[r] - v0 - c;
    float v[CE];
#pragma unroll
    for (int e = 0; e < CE; ++e) {
      if constexpr (EK == EL_F32) v[e] = x[e] * f;
      else v[e] = f16_to_f32(x[e]) * f;
    }
    if (at >= 0 && at < CE) {  // (a rounded exponential less 1 has few bits left where the row is sure)
      const float g = s.row_g[r];
#pragma unroll
      for (int e = 0; e < CE; ++e) v[e] = e == at ? g : v[e];
    }
#pragma unroll
    for (int e = 0; e < CE; ++e) {
      if constexpr (EK == EL_F32) x[e] = v[e];
      else if constexpr (EK == EL_F16) x[e] = f32_to_f16(v[e]);
      else x[e] = f32_to_bf16(v[e]);
    }
    *reinterpret_cast<vec*>(q) = x;
  }
}

template <int EK>
__device__ __forceinline__ uint16_t to_elem(float v) { return EK == EL_F16 ? f32_to_f16(v) : f32_to_bf16(v); }
// What rounding G's value g to the operands' type takes from it.
template <int EK>
__device__ __forceinline__ float g_rest(float g) {
  if constexpr (EK == EL_F32) return 0.0f;
  return g - (EK == EL_F16 ? f16_to_f32(to_elem<EK>(g)) : bf16_to_f32(to_elem<EK>(g)));
}

// dW of few rows (16-bit operands): bound by its stores.  The general product's
// tiles wait for their loads, for LDS and for the queue of the tile before; here
// a wave keeps X's 32 KB rows x 32 CB columns in registers, four waves read the
// next 64 classes of G while they store 64 rows of dW, and no result goes
// through LDS: X's columns are dealt to a pair of 16 x 16 blocks four by four,
// so that a lane holds eight neighbours.  64 x 32003 x 2048 f16 39.6 -> 28.8 us
// (131 MB written; stores alone take 23), 128 x 32000 x 4096 bf16 77.6 -> 59.0,
// 256 105.7 -> 86.2.
// To 128 rows (KB <= 4), what the rounding of G took from a label's value is
// added as products of their own, for the 16 classes that have a label: in a sum
// of so few rows it is most of the error, and it does not average out (30.6 us
// and 62.1).
struct LxDw {
  const uint16_t* g;  // [Rp][ldg]
  const uint16_t* x;  // [Rp][Dp]
  void* dw;
  const int32_t* n;   // rows that count; head[1] behind it
  const int32_t* label;
  const float* row_g;
  int v0;             // class of G's column 0
  int64_t ldg, lddw;
  int Dp, D, classes;
  int per;            // blocks of 64 classes of a workgroup
};

template <int IN, int OUT, int KB, int CB>
__global__ __launch_bounds__(256, 2) void lx_dw_kernel(LxDw a) {
  constexpr int TILE = 32 * KB * 128;  // [32 KB rows][64 columns]
  __shared__ __align__(16) uint8_t smem[2 * TILE];
  __shared__ int lab[32 * KB];        // column of G, -1 behind the last row
  __shared__ uint16_t rest[32 * KB];  // row_g less its rounding, in the operands' type
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int n = a.n[0];
  const float alpha = __int_as_float(a.n[1]);
  const int g16 = lane >> 4, i16 = lane & 15;
  // rows below n of 64 columns from src on, zeros elsewhere (behind `cols` columns too)
  auto fetch = [&](const uint16_t* src, int64_t ld, int cols, u16x8 (&v)[KB]) {
#pragma unroll
    for (int j = 0; j < KB; ++j) {
      const int k = (tid >> 3) + 32 * j, c = (tid & 7) * 8;
      v[j] = k < n && c < cols ? *reinterpret_cast<const u16x8*>(src + k * ld + c) : u16x8{};
    }
  };
  auto put = [&](uint8_t* tile, const u16x8 (&v)[KB]) {
#pragma unroll
    for (int j = 0; j < KB; ++j) {
      const int k = (tid >> 3) + 32 * j;
      *reinterpret_cast<u16x8*>(tile + k * 128 + (((tid & 7) ^ nt_mn_swizzle<16, 2, 8>(k)) * 16)) = v[j];
    }
  };
  // K-rows 8 g16 .. + 7 of a step, eight bytes of each of four lanes a row
  const int row = 8 * g16 + (i16 >> 2), swz = nt_mn_swizzle<16, 2, 8>(row);
  typedef short v4i16 __attribute__((ext_vector_type(4)));
  auto frag = [&](const uint8_t* tile, int kb, int chunk, int half) -> u16x8 {
    const uint8_t* at = tile + (kb * 32 + row) * 128 + ((chunk ^ swz) * 16) + 8 * half;
    const v4i16 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4i16*)at);
    const v4i16 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4i16*)(at + 4 * 128));
    u16x8 f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f[e] = (uint16_t)lo[e];
      f[e + 4] = (uint16_t)hi[e];
    }
    return f;
  };

  constexpr bool REST = KB <= 4;
  if (REST && tid < 32 * KB) {
    lab[tid] = tid < n ? a.label[tid] - a.v0 : -1;
    rest[tid] = tid < n ? to_elem<IN == IN_F16 ? EL_F16 : EL_BF16>(g_rest<IN == IN_F16 ? EL_F16 : EL_BF16>(a.row_g[tid])) : 0;
  }
  const int col0 = blockIdx.x * 128 * CB;                // of the workgroup
  const int blocks = (a.classes + 63) / 64, first = blockIdx.y * a.per;
  const int last = first + a.per < blocks ? first + a.per : blocks;
  u16x8 next[KB];
  fetch(a.g + first * 64, a.ldg, 64, next);
  u16x8 fx[CB][2][KB];
#pragma unroll
  for (int t = 0; t < 2 * CB; ++t) {  // 64 columns each: CB / 2 of them a wave's
    u16x8 v[KB];
    fetch(a.x + col0 + t * 64, a.Dp, a.Dp - col0 - t * 64, v);
    uint8_t* tile = smem + (t & 1) * TILE;
    put(tile, v);
    __syncthreads();
    if (t / (CB / 2) == wave) {
#pragma unroll
      for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int kb = 0; kb < KB; ++kb) fx[t % (CB / 2) * 2 + q][h][kb] = frag(tile, kb, 4 * q + (i16 & 3), h);
    }
  }
  __syncthreads();
  int mine[KB / 2];  // labels of rows lane, lane + 64
#pragma unroll
  for (int i = 0; i < KB / 2; ++i) mine[i] = REST ? lab[i * 64 + lane] : -1;
  for (int b = first; b < last; ++b) {
    const uint8_t* tile = smem + (b & 1) * TILE;
    put(smem + (b & 1) * TILE, next);
    __syncthreads();  // (the other tile's readers are behind the barrier before)
    if (b + 1 < last) fetch(a.g + (b + 1) * 64, a.ldg, 64, next);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      u16x8 fg[KB];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) fg[kb] = frag(tile, kb, 2 * j + ((i16 >> 1) & 1), i16 & 1);
      const int v = b * 64 + j * 16 + i16;
      u16x8 fr[REST ? KB : 1];
      bool has = false;  // a label among these 16 classes
      if constexpr (REST) {
#pragma unroll
        for (int i = 0; i < KB / 2; ++i) has |= (mine[i] >> 4) == b * 4 + j;
        has = __any(has);
      }
      if (REST && has) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int k = kb * 32 + 8 * g16 + e;
            fr[kb][e] = lab[k] == v ? rest[k] : 0;
          }
      }
#pragma unroll
      for (int p = 0; p < CB; ++p) {
        floatx4 acc[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          acc[h] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int kb = 0; kb < KB; ++kb)
            acc[h] = mfma16<IN>(reinterpret_cast<const uint16_t*>(&fx[p][h][kb]),
                                reinterpret_cast<const uint16_t*>(&fg[kb]), acc[h]);
          if (REST && has) {
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
              acc[h] = mfma16<IN>(reinterpret_cast<const uint16_t*>(&fx[p][h][kb]),
                                  reinterpret_cast<const uint16_t*>(&fr[kb]), acc[h]);
          }
        }
        const int c = col0 + wave * 32 * CB + p * 32 + 8 * g16;
        if (v >= a.classes || c >= a.D) continue;
        float o[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = acc[e >> 2][e & 3] * alpha;
        if constexpr (OUT == OUT_F32) {
          float* q = (float*)a.dw + v * a.lddw + c;
          if (c + 8 <= a.D) {
            reinterpret_cast<f32x4_a4*>(q)[0] = f32x4_a4{o[0], o[1], o[2], o[3]};
            reinterpret_cast<f32x4_a4*>(q)[1] = f32x4_a4{o[4], o[5], o[6], o[7]};
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (c + e < a.D) q[e] = o[e];
          }
        } else {
          uint16_t* q = (uint16_t*)a.dw + v * a.lddw + c;
          u16x8_a2 r;
#pragma unroll
          for (int e = 0; e < 8; ++e) r[e] = OUT == OUT_F16 ? f32_to_f16(o[e]) : f32_to_bf16(o[e]);
          if (c + 8 <= a.D) {
            *reinterpret_cast<u16x8_a2*>(q) = r;
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (c + e < a.D) q[e] = r[e];
          }
        }
      }
    }
  }
}

// Columns of a workgroup and blocks of 64 classes that each has, for R <= 256 rows.
constexpr int kFewRows = 128;
int lx_dw_cols(int64_t R) { return R <= kFewRows ? 512 : 256; }
int lx_dw_blocks(int64_t R, int64_t classes, int64_t D) {
  const int64_t gx = (D + lx_dw_cols(R) - 1) / lx_dw_cols(R), blocks = (classes + 63) / 64;
  const int64_t share = std::max<int64_t>(1, 512 / gx);  // two workgroups run on a CU
  return (int)((blocks + share - 1) / share);
}
// 16-bit operands: always to 128 rows; to 256 where each workgroup has three
// blocks or more, over which X's loads are spread (10007 x 2048 21.6 us against
// the product's 25.8, but 16384 x 1024 19.0 against 17.4).
bool lx_dw_fits(int64_t R, int64_t classes, int64_t D) {
  return R <= kFewRows || (R <= 256 && lx_dw_blocks(R, classes, D) >= 3);
}

template <int IN, int OUT>
Status lx_dw(LxDw a, int64_t R, hipStream_t s) {
  const int cols = lx_dw_cols(R), blocks = (a.classes + 63) / 64;
  a.per = lx_dw_blocks(R, a.classes, a.D);
  const dim3 grid((a.D + cols - 1) / cols, (blocks + a.per - 1) / a.per);
  if (R <= kFewRows / 2) lx_dw_kernel<IN, OUT, 2, 4><<<grid, 256, 0, s>>>(a);
  else if (R <= kFewRows) lx_dw_kernel<IN, OUT, 4, 4><<<grid, 256, 0, s>>>(a);
  else lx_dw_kernel<IN, OUT, 8, 2><<<grid, 256, 0, s>>>(a);
  return launch_status("linear_xent_dw");
}

// dX from its slabs: head[1] times their sum, in order, to the row it came from.
// rest: and what the rounding of G took from the label's value, from W's row.
template <int EK>
__global__ __launch_bounds__(256) void lx_finish_kernel(LxRows s, int direct, int k_piece, int bm, int64_t ld, int D,
                                                        void* dx, int64_t lddx, const void* rest, int64_t ldw) {
  const int n = s.head[0], shares = s.head[4];
  if (direct && shares == 1) return;  // (stored by the product itself)
  const int k_share = lx_share_k(k_piece, shares), slabs = lx_slabs(k_piece, k_share);
  const int64_t stride = (int64_t)((n + bm - 1) / bm * bm) * ld;
  const float alpha = __int_as_float(s.head[1]);
  const int c = (blockIdx.x * 256 + threadIdx.x) * 4;
  if (c >= D) return;
  for (int r = blockIdx.y; r < n; r += gridDim.y) {
    const float* q = s.slab + (int64_t)r * ld + c;
    f32x4 v{0.0f, 0.0f, 0.0f, 0.0f};
    int k = 0;
    for (; k + 8 <= slabs; k += 8) {
      f32x4 x[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) x[u] = *reinterpret_cast<const f32x4*>(q + (k + u) * stride);
#pragma unroll
      for (int u = 0; u < 8; ++u) v += x[u];
    }
    for (; k < slabs; ++k) v += *reinterpret_cast<const f32x4*>(q + k * stride);
    const int64_t at = (int64_t)s.idx[r] * lddx + c;
    const float g = rest ? g_rest<EK>(s.row_g[r]) : 0.0f;
    const int64_t w_at = (int64_t)s.label[r] * ldw + c;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (c + e < D) {
        float x = v[e];
        if (rest) x = fmaf(g, elem_f32<EK>(rest, w_at + e), x);
        x *= alpha;
        if constexpr (EK == EL_F32) ((float*)dx)[at + e] = x;
        else ((uint16_t*)dx)[at + e] = EK == EL_F16 ? f32_to_f16(x) : f32_to_bf16(x);
      }
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
struct LxCall {
  const TensorDesc *x, *w, *labels, *rw, *loss, *dx, *dw, *row_loss, *scratch;
  int ek;  // ElemKind of X and W
  int64_t R, V, D, ldx, ldw, lddx, lddw;
};

template <int IN, int OUT, int ACT, int BM, int BN, int WM, int WN, bool AKC, bool BKC, int S>
Status lx_gemm_as(const NTParams& q, int64_t rows, int64_t cols, hipStream_t s) {
  NTParams p = q;
  p.tiles_m = (int)((rows + BM - 1) / BM);
  p.tiles_n = (int)((cols + BN - 1) / BN);
  const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n;
  if (tiles == 0) return Status::Ok;
  if (tiles > INT32_MAX) return Status::InvalidArgument;
  unsigned grid = (unsigned)tiles;
  if constexpr (ACT == ACT_LX_SLAB) {
    grid = (unsigned)lx_slots(BM, IN == IN_F32);  // they loop over the tiles' shares
  } else if constexpr (nt_persistent(BM, BN, WM, WN)) {
    const int ncu = device_cu_count();
    if (ncu > 0 && ncu % 8 == 0 && grid > (unsigned)ncu) grid = (unsigned)ncu;
  }
  gemm_nt_kernel<IN, OUT, ACT, BM, BN, WM, WN, AKC, BKC, S><<<grid, 64 * WM * WN, 0, s>>>(p);
  return launch_status("linear_xent");
}

// rows x cols of the product in tiles of bm rows.
template <int IN, int OUT, int ACT, bool AKC, bool BKC>
Status lx_gemm(const NTParams& p, int bm, int64_t rows, int64_t cols, hipStream_t s) {
  if constexpr (IN == IN_F32) {
    if constexpr (AKC) {
      if (bm == 32) return lx_gemm_as<IN, OUT, ACT, 32, 128, 1, 4, AKC, BKC, 2>(p, rows, cols, s);
    }
    if (bm == 64) return lx_gemm_as<IN, OUT, ACT, 64, 64, 2, 2, AKC, BKC, 2>(p, rows, cols, s);
  } else {
    // Both operands K-contiguous (logits) and long K: four waves of 128 x 128, which read half the LDS bytes a
    // product (8192 x 32000 x 4096 bf16 1719 -> 1656 us, 4096 x 32000 x 4096 897 -> 868; x 1024 300, 327).
    if constexpr (AKC && BKC) {
      if (bm == 256 && !lx_tiles_loop(bm, false, p.K)) return lx_gemm_as<IN, OUT, ACT, 256, 256, 2, 2, AKC, BKC, 2>(p, rows, cols, s);
    }
    if (bm == 256) return lx_gemm_as<IN, OUT, ACT, 256, 256, 2, 4, AKC, BKC, 2>(p, rows, cols, s);
    if constexpr (AKC) {
      if (bm == 32) return lx_gemm_as<IN, OUT, ACT, 32, 128, 1, 4, AKC, BKC, 4>(p, rows, cols, s);
      if (bm == 64) return lx_gemm_as<IN, OUT, ACT, 64, 128, 1, 4, AKC, BKC, 4>(p, rows, cols, s);
    }
  }
  return lx_gemm_as<IN, OUT, ACT, 128, 128, 2, 2, AKC, BKC, 2>(p, rows, cols, s);
}

template <int IN, int EK>
Status lx_run(const LxCall& c, const LxPlan& pl, hipStream_t s) {
  constexpr int ES = IN == IN_F32 ? 4 : 2;
  constexpr int OUT = IN == IN_F32 ? OUT_F32 : IN == IN_F16 ? OUT_F16 : OUT_BF16;
  uint8_t* base = (uint8_t*)(((uintptr_t)c.scratch->data + 255) & ~(uintptr_t)255);
  LxRows rw{};
  rw.head = (int32_t*)base;
  int32_t* arr = (int32_t*)(base + 256);
  rw.idx = arr;
  rw.label = arr + pl.Rp;
  rw.weight = (float*)arr + 2 * pl.Rp;
  rw.row_g = (float*)arr + 3 * pl.Rp;
  rw.zlab = (float*)arr + 4 * pl.Rp;
  rw.row_max = (float*)arr + 5 * pl.Rp;
  rw.row_f = (float*)arr + 6 * pl.Rp;
  rw.row_loss = (float*)arr + 7 * pl.Rp;
  rw.stats = (float2*)(base + pl.stats_off);
  rw.xc = base + pl.xc_off;
  rw.slab = (float*)(base + pl.slab_off);
  rw.wpad = base + pl.wpad_off;
  rw.g = base + pl.g_off;
  const float* alpha = (const float*)(rw.head + 1);
  const int R = (int)c.R, V = (int)c.V, D = (int)c.D, Dp = (int)pl.Dp;
  const int top = IN == IN_F16 ? 13 : 0;  // G of at most 2^13 in f16
  float* row_loss = (float*)c.row_loss->data;

  const bool grad = c.dx != nullptr;
  const int tn_dx = lx_tile_cols(pl.bm_dx, IN == IN_F32);
  const LxParts pt = lx_parts(pl, c.V, grad);
  const LxShares sh{pl.bm_dx, grad ? (D + tn_dx - 1) / tn_dx : 0, lx_slots(pl.bm_dx, IN == IN_F32),
                    (int)pt.longest(), (int)std::min<int64_t>(pl.slab_rows, INT32_MAX)};
  const LxCopy cx{c.x->data, rw.xc, grad ? c.dx->data : nullptr, row_loss, c.ldx, c.lddx, D, Dp};
  const int32_t* labels = (const int32_t*)c.labels->data;
  const float* weight = c.rw ? (const float*)c.rw->data : nullptr;
  if (R <= kCountedByAll) {
    const int per = std::max(1, (R + 255) / 256);
    const unsigned groups = R > 0 ? (R + per - 1) / per : 1;
    if (R <= 1024) lx_rows_kernel<ES, 1><<<groups, 1024, 0, s>>>(labels, weight, R, V, top, rw, sh, cx, per, nullptr);
    else lx_rows_kernel<ES, 4><<<groups, 1024, 0, s>>>(labels, weight, R, V, top, rw, sh, cx, per, nullptr);
  } else {
    int32_t* pos = (int32_t*)rw.row_loss;  // (written by lx_stats_kernel)
    lx_rows_kernel<ES, 16><<<1, 1024, 0, s>>>(labels, weight, R, V, top, rw, sh, cx, 0, pos);
    lx_copy_rows_kernel<ES><<<(R + 3) / 4, 256, 0, s>>>(cx, R, pos);
  }
  Status st = launch_status("linear_xent_rows");
  if (st != Status::Ok) return st;

  // W's rows of the classes v0 .. v0 + cols, in place or copied (unless the copy is there)
  int64_t copied = -1;
  auto weights = [&](NTParams& p, int64_t v0, int64_t cols) {
    const uint8_t* w = (const uint8_t*)c.w->data + v0 * c.ldw * ES;
    if (pl.direct) {
      p.B = w;
      p.ldb = c.ldw;
    } else {
      if (copied != v0)
        lx_copy_rows_kernel<ES><<<(unsigned)((cols + 3) / 4), 256, 0, s>>>(
            LxCopy{w, rw.wpad, nullptr, nullptr, c.ldw, 0, D, Dp}, (int)cols, nullptr);
      copied = v0;
      p.B = rw.wpad;
      p.ldb = Dp;
    }
  };
  struct Part {  // classes v0 .. v0 + cols and their G
    int64_t v0, cols;
    void* g;
    int64_t ldg;
  };
  auto logits = [&](int64_t v0, int64_t cols, const Part& keep) {
    NTParams p{};
    weights(p, v0, cols);
    p.A = rw.xc;
    p.lda = Dp;
    p.C = keep.g;
    p.ldc = keep.ldg;
    p.M = R;
    p.N = (int)cols;
    p.K = pl.direct ? D : Dp;
    p.lx.n = rw.head;
    p.lx.a_mn = (int)pl.Rp;
    p.lx.b_mn = (int)cols;
    p.lx.v0 = (int)v0;
    p.lx.label = rw.label;
    p.lx.zlab = rw.zlab;
    p.lx.stats = rw.stats;
    p.lx.stats_ld = pl.Rp;
    p.lx.row_max = rw.row_max;
    p.lx.row_f = rw.row_f;
    p.lx.row_g = rw.row_g;
    return p;
  };
  const int64_t last = pt.last, parts = pt.count;
  const int kept = pt.kept;
  auto part = [&](int64_t k) -> Part {
    const LxPart q = pt.at(k);
    if (k >= kept - 1) return {q.v0, q.cols, rw.g, pl.piece};
    const uintptr_t at = (uintptr_t)c.dw->data + pl.held * D * (dt(*c.dw) == DType::kF32 ? 4 : 2);
    return {q.v0, q.cols, (void*)((at + 255) & ~(uintptr_t)255), pl.held};
  };
  auto stats = [&](const Part& q, int64_t cols, int64_t keep_from) {
    NTParams p = logits(q.v0, cols, q);
    p.lx.keep_from = (int)keep_from;
    return lx_gemm<IN, OUT, ACT_LX_STATS, true, true>(p, pl.bm, R, cols, s);
  };
  if (pl.direct) {  // W read in place: all classes behind the held ones at once
    if (pl.held > 0 && (st = stats(part(0), pl.held, 0)) != Status::Ok) return st;
    st = stats({pl.held, 0, rw.g, pl.piece}, c.V - pl.held, last - pl.held);
    if (st != Status::Ok) return st;
  } else {
    for (int64_t k = 0; k < parts; ++k) {
      const Part q = part(k);
      st = stats(q, q.cols, k < kept ? 0 : INT32_MAX);
      if (st != Status::Ok) return st;
    }
  }
  float* loss = (float*)c.loss->data;
  lx_stats_kernel<<<R > 0 ? (R + 63) / 64 : 1, 1024, 0, s>>>(rw, (int)((c.V + pl.bn - 1) / pl.bn), pl.Rp, weight != nullptr,
                                                             row_loss, R <= 64 ? loss : nullptr);
  if (R > 64) lx_loss_kernel<<<1, 1024, 0, s>>>(rw, loss);
  st = launch_status("linear_xent_stats");
  if (st != Status::Ok || !grad) return st;

  // Few rows of 16 bits: their labels' values of G count in full (lx_dw_kernel, lx_finish_kernel).
  const bool few = IN != IN_F32 && R <= kFewRows;
  const bool direct = parts == 1 && !few;  // dX needs no slab unless its K is shared
  int64_t k_before = 0;
  for (int64_t k = 0; k < parts; ++k) {
    const Part q = part(k);
    const int64_t v0 = q.v0, cols = q.cols;
    if (k < kept) {
      if (R > 0) {
        const int64_t width = lx_up_to(cols, pl.bn);
        const unsigned gx = (unsigned)((width + 256 * (16 / ES) - 1) / (256 * (16 / ES)));
        const unsigned gy = (unsigned)std::min<int64_t>(R, 32768);
        if (pl.bn == 64)
          lx_scale_kernel<EK, 64><<<dim3(gx, gy), 256, 0, s>>>(rw, q.g, q.ldg, (int)width, (int)v0, pl.Rp);
        else if (pl.bn == 256)
          lx_scale_kernel<EK, 256><<<dim3(gx, gy), 256, 0, s>>>(rw, q.g, q.ldg, (int)width, (int)v0, pl.Rp);
        else
          lx_scale_kernel<EK, 128><<<dim3(gx, gy), 256, 0, s>>>(rw, q.g, q.ldg, (int)width, (int)v0, pl.Rp);
      }
    } else {
      NTParams p = logits(v0, cols, q);
      st = lx_gemm<IN, OUT, ACT_LX_GRAD, true, true>(p, pl.bm, R, cols, s);
      if (st != Status::Ok) return st;
    }
    if (c.dw) {
      NTParams p{};
      p.A = q.g;
      p.lda = q.ldg;
      p.B = rw.xc;
      p.ldb = Dp;
      p.M = (int)cols;
      p.N = D;
      p.K = R;
      p.ldc = c.lddw;
      p.lx.n = rw.head;
      p.lx.rows_are_k = 1;
      p.lx.a_mn = (int)q.ldg;
      p.lx.b_mn = Dp;
      p.lx.alpha = alpha;
      const bool f32 = dt(*c.dw) == DType::kF32;
      const int ob = f32 ? 4 : 2;
      p.C = (uint8_t*)c.dw->data + v0 * c.lddw * ob;
      p.lx.vec = aligned(c.dw->data, 16) && c.lddw * ob % 16 == 0;
      const int bm = lx_tile_rows(std::max<int64_t>(cols, 129), c.D, IN == IN_F32);
      const bool dw_few = IN != IN_F32 && lx_dw_fits(R, cols, D);
      if constexpr (IN != IN_F32) {
        if (dw_few) {
          const LxDw a{(const uint16_t*)q.g, (const uint16_t*)rw.xc, p.C, rw.head, rw.label, rw.row_g,
                       (int)v0, q.ldg, c.lddw, Dp, D, (int)cols, 0};
          st = f32 ? lx_dw<IN, OUT_F32>(a, R, s) : lx_dw<IN, OUT>(a, R, s);
        }
      }
      if (dw_few)
        ;
      else if (f32)
        st = lx_gemm<IN, OUT_F32, ACT_LX_OUT, false, false>(p, bm, cols, D, s);
      else
        st = lx_gemm<IN, OUT, ACT_LX_OUT, false, false>(p, bm, cols, D, s);
      if (st != Status::Ok) return st;
    }
    if (R > 0) {
      NTParams p{};
      weights(p, v0, cols);
      p.A = q.g;
      p.lda = q.ldg;
      p.M = R;
      p.N = D;
      p.K = (int)cols;
      p.lx.n = rw.head;
      p.lx.a_mn = (int)pl.Rp;
      p.lx.b_mn = pl.direct ? D : Dp;
      p.lx.shares = rw.head + 4;
      if (direct) {
        p.lx.direct = c.dx->data;
        p.lx.ld_direct = c.lddx;
        p.lx.alpha = alpha;
        p.lx.row_map = rw.idx;
        p.lx.vec = aligned(c.dx->data, 16) && c.lddx * ES % 16 == 0;
      }
      p.C = rw.slab;
      p.ldc = Dp;
      p.lx.k_piece = sh.k_piece;
      p.lx.k_before = (int)k_before;
      k_before = std::max(k_before, cols);
      st = lx_gemm<IN, OUT, ACT_LX_SLAB, true, false>(p, pl.bm_dx, R, D, s);
      if (st != Status::Ok) return st;
    }
  }
  if (R > 0) {
    const unsigned gx = (unsigned)((D + 1023) / 1024), gy = (unsigned)std::min<int64_t>(R, 32768);
    lx_finish_kernel<EK><<<dim3(gx, gy), 256, 0, s>>>(rw, direct, sh.k_piece, pl.bm_dx, Dp, D, c.dx->data, c.lddx,
                                                      few ? c.w->data : nullptr, c.ldw);
    return launch_status("linear_xent_finish");
  }
  return Status::Ok;
}

// Whether tiles read W with 16-byte loads.
bool lx_in_place(const TensorDesc& w, int64_t ldw, int64_t es) {
  const int64_t V = w.shape[0], D = w.shape[1];
  return D * es % 16 == 0 && aligned(w.data, 16) && ldw * es % 16 == 0 && (V == 1 || ldw >= D) &&
         ldw < INT32_MAX / (256 * es);
}

// X, W, labels [, weights] -> loss, row loss, scratch | loss, dX, row loss,
// scratch | loss, dX, dW, row loss, scratch.
bool lx_read(const TensorDesc* in, int ni, const TensorDesc* out, int no, LxCall* pc, LxPlan* pl) {
  if (!in || !out || (ni != 3 && ni != 4) || no < 3 || no > 5) return false;
  LxCall c{};
  c.x = &in[0];
  c.w = &in[1];
  c.labels = &in[2];
  c.rw = ni == 4 ? &in[3] : nullptr;
  c.loss = &out[0];
  c.dx = no >= 4 ? &out[1] : nullptr;
  c.dw = no == 5 ? &out[2] : nullptr;
  c.row_loss = &out[no - 2];
  c.scratch = &out[no - 1];
  int wk;
  if (!elem_kind(*c.x, &c.ek) || !elem_kind(*c.w, &wk) || wk != c.ek) return false;
  if (!matrix_ld(*c.x, false, &c.ldx) || !matrix_ld(*c.w, false, &c.ldw)) return false;
  c.R = c.x->shape[0];
  c.D = c.x->shape[1];
  c.V = c.w->shape[0];
  if (c.w->shape[1] != c.D || c.V < 1 || c.D < 1) return false;
  if (!vector_of(*c.labels, DType::kI32, c.R)) return false;
  if (c.rw && !vector_of(*c.rw, DType::kF32, c.R)) return false;
  if (!vector_of(*c.loss, DType::kF32, 1) || !vector_of(*c.row_loss, DType::kF32, c.R)) return false;
  if (dt(*c.scratch) != DType::kF32 || c.scratch->rank != 1 || (c.scratch->shape[0] > 1 && c.scratch->stride[0] != 1))
    return false;
  auto grad_of = [](const TensorDesc& g, const TensorDesc& of, int64_t* ld, bool f32_too) {
    return matrix_ld(g, true, ld) && same_shape(g, of) && (dt(g) == dt(of) || (f32_too && dt(g) == DType::kF32));
  };
  if (c.dx && !grad_of(*c.dx, *c.x, &c.lddx, false)) return false;
  if (c.dw && !grad_of(*c.dw, *c.w, &c.lddw, true)) return false;
  if (any_overlap(in, ni, out, no)) return false;
  const bool f32 = c.ek == EL_F32, direct = lx_in_place(*c.w, c.ldw, f32 ? 4 : 2);
  if (!lx_plan(c.R, c.V, c.D, c.ldw, direct, f32, c.dx != nullptr, 0, c.scratch->shape[0] * 4, pl)) return false;
  if (c.dw && (c.V == 1 || c.lddw == c.D)) pl->held = lx_held(*pl, c.V, c.D, c.ldw, dt(*c.dw) == DType::kF32 ? 4 : 2);
  if (pc) *pc = c;
  return true;
}

bool lx_sup(const TensorDesc* in, int ni, const TensorDesc* out, int no, const void*) {
  LxPlan pl;
  return lx_read(in, ni, out, no, nullptr, &pl);
}

Status lx_launch(const TensorDesc* in, int ni, TensorDesc* out, int no, const void*, void*, size_t, void* stream) {
  LxCall c;
  LxPlan pl;
  if (!lx_read(in, ni, out, no, &c, &pl)) return Status::InvalidArgument;
  for (int k = 0; k < ni; ++k)
    if (no_memory(in[k])) return Status::InvalidArgument;
  for (int k = 0; k < no; ++k)
    if (no_memory(out[k])) return Status::InvalidArgument;
  hipStream_t s = as_stream(stream);
  if (c.ek == EL_F32) return lx_run<IN_F32, EL_F32>(c, pl, s);
  if (c.ek == EL_F16) return lx_run<IN_F16, EL_F16>(c, pl, s);
  return lx_run<IN_BF16, EL_BF16>(c, pl, s);
}

size_t no_workspace(const TensorDesc*, int, const void*) { return 0; }

}  // namespace

KernelVariant make_linear_xent_variant() {
  KernelVariant v;
  v.name = "linear_xent";
  v.launch = lx_launch;
  v.supported = lx_sup;
  v.query_workspace = no_workspace;
  return v;
}

}  // namespace aicf::hip

using namespace aicf::hip;

extern "C" int64_t aicf_linear_xent_scratch(int64_t rows, int64_t classes, int64_t dim, int32_t dtype,
                                            int32_t gradients, int64_t piece) {
  if (rows < 0 || classes < 1 || dim < 1 ||
      (dtype != AICF_DTYPE_F32 && dtype != AICF_DTYPE_F16 && dtype != AICF_DTYPE_BF16))
    return -1;
  const bool f32 = dtype == AICF_DTYPE_F32;
  LxPlan p;
  if (rows > INT32_MAX || classes > INT32_MAX || dim > INT32_MAX ||
      !lx_plan(rows, classes, dim, dim, dim * (f32 ? 4 : 2) % 16 == 0, f32, gradients != 0, piece, -1, &p))
    return -1;
  return p.bytes;
}

extern "C" int64_t aicf_linear_xent_scratch_for(int64_t rows, const aicf_tensor_desc* w, int32_t gradients,
                                                int64_t piece) {
  int ek;
  int64_t ldw;
  if (!w || !elem_kind(*w, &ek) || !matrix_ld(*w, false, &ldw)) return -1;
  const int64_t V = w->shape[0], D = w->shape[1];
  if (rows < 0 || V < 1 || D < 1 || rows > INT32_MAX || V > INT32_MAX || D > INT32_MAX) return -1;
  const bool f32 = ek == EL_F32;
  LxPlan p;
  if (!lx_plan(rows, V, D, ldw, lx_in_place(*w, ldw, f32 ? 4 : 2), f32, gradients != 0, piece, -1, &p)) return -1;
  return p.bytes;
}
