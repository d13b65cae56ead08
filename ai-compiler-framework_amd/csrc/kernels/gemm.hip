// GEMM and GEMM + fused epilogue for gfx950 on the MFMA matrix cores.
//
//   C[M,N] = epi( op(A)[M,K] . op(B)[K,N] )
//
// Reference contracts:
//   Gemm          src/backends/cuda/ops/gemm/launcher.cu:41-70 (attrs <ii> transA,
//                 transB under schema 0 or GEMM), :75-148 (2-D views, checks),
//                 :342-359 (f16 path needs a row-major contiguous C)
//   GemmEpilogue  src/backends/cuda/ops/gemm_epilogue/launcher.cu:49-80 (attrs
//                 <iii> transA, transB, relu under schema 0 or GPEL, relu
//                 default 1), :153-193 (checks: bias rank 1, length N)
//                 plus the executor's GEPI layout <iii> transA, transB, kind
//                 (core_v2/exec.py:211-252), honoured here as documented.
//
// Kernel design (one templated kernel, all dtypes):
//   * workgroup tile BM x BN x BK, WM x WN waves, each wave owns a
//     (BM/WM) x (BN/WN) block of 32x32 MFMA tiles with fp32 accumulators;
//   * 16-bit inputs use v_mfma_f32_32x32x16_{bf16,f16}, fp32 inputs use
//     v_mfma_f32_32x32x2f32 (true fp32 products, no reduced-precision path);
//   * A and B tiles live in LDS as [rows][BK] with K contiguous; 16-byte
//     chunks of a row are XOR-swizzled by (row mod chunks-per-row) so the
//     fragment reads of 32 consecutive rows spread over all banks;
//   * operands whose K stride is 1 are copied with 16-byte loads; operands
//     whose M/N stride is 1 (transposed views) are loaded 16 bytes along
//     M/N and transposed on the LDS write; anything else is gathered per
//     element;
//   * two LDS buffers: the global loads of tile k+1 are in flight while the
//     MFMAs of tile k run, with one barrier per K step;
//   * workgroup ids are remapped so that consecutive tiles of one XCD share
//     A rows (grouped column-major raster per XCD).
#include <type_traits>
#include <utility>

#include "../common/gemm_nt.hpp"
#include "../common/smallstep.hpp"

namespace aicf::hip {

namespace {

// XOR swizzle of the 16-byte chunk index inside one LDS row.
template <int NCH>
__device__ __forceinline__ int swz(int row, int chunk) {
  return chunk ^ (row & (NCH - 1));
}

// Loads one operand tile (ROWS x BK, rows along M or N) from global memory
// into registers, then writes it to LDS.  `rs` steps along the tile rows
// (M or N), `cs` along K.
template <int IN, int ROWS, int BK, int THREADS>
struct TileLoader {
  typedef typename InTraits<IN>::T T;
  static constexpr int CE = InTraits<IN>::CE;
  static constexpr int NCH = BK / CE;                    // chunks per LDS row
  static constexpr int CHUNKS = ROWS * BK / CE;          // 16-byte chunks per tile
  static constexpr int PER_THREAD = (CHUNKS + THREADS - 1) / THREADS;
  typedef T vec __attribute__((ext_vector_type(CE)));
  vec r[PER_THREAD];

  // mode LD_KCONTIG: chunk c covers row c / NCH, k chunk c % NCH.
  // mode LD_MNCONTIG: chunk c covers k row c / (ROWS/CE), row chunk c % (ROWS/CE).
  __device__ void load(const T* __restrict__ g, int mode, int64_t row0, int64_t rows_total,
                       int64_t k0, int64_t K, int64_t rs, int64_t cs, bool vec_ok) {
    const int t = threadIdx.x;
#pragma unroll
    for (int i = 0; i < PER_THREAD; ++i) {
      const int c = t + i * THREADS;
      vec v;
#pragma unroll
      for (int e = 0; e < CE; ++e) v[e] = T(0);
      if (c < CHUNKS) {
        if (mode == LD_KCONTIG) {
          const int row = c / NCH, kc = c % NCH;
          const int64_t gr = row0 + row, gk = k0 + (int64_t)kc * CE;
          if (gr < rows_total) {
            if (vec_ok && gk + CE <= K) {
              v = *reinterpret_cast<const vec*>(g + gr * rs + gk);
            } else {
#pragma unroll
              for (int e = 0; e < CE; ++e)
                if (gk + e < K) v[e] = g[gr * rs + (gk + e) * cs];
            }
          }
        } else {
          constexpr int RCH = ROWS / CE;
          const int kr = c / RCH, rc = c % RCH;
          const int64_t gk = k0 + kr, gr = row0 + (int64_t)rc * CE;
          if (gk < K) {
            if (mode == LD_MNCONTIG && vec_ok && gr + CE <= rows_total) {
              v = *reinterpret_cast<const vec*>(g + gk * cs + gr);
            } else {
#pragma unroll
              for (int e = 0; e < CE; ++e)
                if (gr + e < rows_total) v[e] = g[(gr + e) * rs + gk * cs];
            }
          }
        }
      }
      r[i] = v;
    }
  }

  __device__ void store(T* __restrict__ lds, int mode) const {
    const int t = threadIdx.x;
#pragma unroll
    for (int i = 0; i < PER_THREAD; ++i) {
      const int c = t + i * THREADS;
      if (c >= CHUNKS) continue;
      if (mode == LD_KCONTIG) {
        const int row = c / NCH, kc = c % NCH;
        *reinterpret_cast<vec*>(lds + row * BK + swz<NCH>(row, kc) * CE) = r[i];
      } else {
        constexpr int RCH = ROWS / CE;
        const int kr = c / RCH, rc = c % RCH;
        const int kc = kr / CE, ke = kr % CE;
#pragma unroll
        for (int e = 0; e < CE; ++e) {
          const int row = rc * CE + e;
          lds[row * BK + swz<NCH>(row, kc) * CE + ke] = r[i][e];
        }
      }
    }
  }
};

__device__ __forceinline__ void tile_coords(int tiles_m, int tiles_n, int& tm, int& tn) {
  tile_coords_of(blockIdx.x, tiles_m, tiles_n, tm, tn);
}

template <int IN, int OUT, int BM, int BN, int BK, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void gemm_mfma_kernel(GemmParams p) {
  typedef typename InTraits<IN>::T T;
  constexpr int THREADS = 64 * WM * WN;
  constexpr int CE = InTraits<IN>::CE;
  constexpr int KPM = InTraits<IN>::KPM;
  constexpr int EPL = InTraits<IN>::EPL;
  constexpr int NCH = BK / CE;
  constexpr int WTM = BM / WM, WTN = BN / WN;
  constexpr int TM = WTM / 32, TN = WTN / 32;
  static_assert(TM >= 1 && TN >= 1, "wave tile must hold a 32x32 block");

  __shared__ __attribute__((aligned(16))) T lds_a[2][BM * BK];
  __shared__ __attribute__((aligned(16))) T lds_b[2][BN * BK];

  int tm_i, tn_i;
  tile_coords(p.tiles_m, p.tiles_n, tm_i, tn_i);
  const int64_t m0 = (int64_t)tm_i * BM, n0 = (int64_t)tn_i * BN;

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = wave / WN, wn = wave % WN;

  const T* A = (const T*)p.A;
  const T* B = (const T*)p.B;
  // vector loads need 16-byte aligned rows and base
  const int a_lead = p.a_mode == LD_KCONTIG ? 0 : 1;
  const bool a_vec = (p.a_mode != LD_GATHER) && ((uintptr_t)A % 16 == 0) &&
                     (((a_lead == 0 ? p.a_rs : p.a_cs) * (int64_t)sizeof(T)) % 16 == 0);
  const bool b_vec = (p.b_mode != LD_GATHER) && ((uintptr_t)B % 16 == 0) &&
                     (((p.b_mode == LD_KCONTIG ? p.b_cs : p.b_rs) * (int64_t)sizeof(T)) % 16 == 0);

  TileLoader<IN, BM, BK, THREADS> la;
  TileLoader<IN, BN, BK, THREADS> lb;
  // A tile rows are M (row stride a_rs, k stride a_cs); B tile rows are N
  // (row stride b_cs, k stride b_rs).
  floatx16 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;

  const int nk = (int)((p.K + BK - 1) / BK);
  la.load(A, p.a_mode, m0, p.M, 0, p.K, p.a_rs, p.a_cs, a_vec);
  lb.load(B, p.b_mode, n0, p.N, 0, p.K, p.b_cs, p.b_rs, b_vec);
  la.store(lds_a[0], p.a_mode);
  lb.store(lds_b[0], p.b_mode);
  __syncthreads();

  for (int kt = 0; kt < nk; ++kt) {
    const int cur = kt & 1;
    if (kt + 1 < nk) {
      la.load(A, p.a_mode, m0, p.M, (int64_t)(kt + 1) * BK, p.K, p.a_rs, p.a_cs, a_vec);
      lb.load(B, p.b_mode, n0, p.N, (int64_t)(kt + 1) * BK, p.K, p.b_cs, p.b_rs, b_vec);
    }
    const T* sa = lds_a[cur];
    const T* sb = lds_b[cur];
#pragma unroll
    for (int ks = 0; ks < BK / KPM; ++ks) {
      // fragment k position of this lane inside the tile
      const int k = ks * KPM + (lane >> 5) * EPL;
      const int kc = k / CE, ke = k % CE;
      T fa[TM][EPL], fb[TN][EPL];
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const int row = wm * WTM + i * 32 + (lane & 31);
        const T* src = sa + row * BK + swz<NCH>(row, kc) * CE + ke;
        if constexpr (EPL == 8) {
          *reinterpret_cast<u16x8*>(fa[i]) = *reinterpret_cast<const u16x8*>(src);
        } else {
          fa[i][0] = src[0];
        }
      }
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const int row = wn * WTN + j * 32 + (lane & 31);
        const T* src = sb + row * BK + swz<NCH>(row, kc) * CE + ke;
        if constexpr (EPL == 8) {
          *reinterpret_cast<u16x8*>(fb[j]) = *reinterpret_cast<const u16x8*>(src);
        } else {
          fb[j][0] = src[0];
        }
      }
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = mfma32<IN>(fa[i], fb[j], acc[i][j]);
    }
    if (kt + 1 < nk) {
      la.store(lds_a[cur ^ 1], p.a_mode);
      lb.store(lds_b[cur ^ 1], p.b_mode);
    }
    __syncthreads();
  }

  // Epilogue.  Accumulator r of lane l in tile (i, j) holds
  // row 8*(r/4) + 4*(l/32) + r%4 and column l%32 of that 32x32 block.
#pragma unroll
  for (int i = 0; i < TM; ++i) {
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int64_t n = n0 + wn * WTN + j * 32 + (lane & 31);
      if (n >= p.N) continue;
      float bv = 0.0f;
      if (p.bias) {
        bv = p.bias_f32 ? ((const float*)p.bias)[n * p.bias_s] : load_out<OUT>(p.bias, n * p.bias_s);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int64_t m = m0 + wm * WTM + i * 32 + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3);
        if (m >= p.M) continue;
        float v = acc[i][j][r];
        if (p.act == ACT_DGELU) {
          v = v * gelu_tanh_grad_f(load_out<OUT>(p.aux, m * p.aux_rs + n));
        } else {
          v += bv;
          if (p.act == ACT_RELU) {
            v = v > 0.0f ? v : 0.0f;
          } else if (p.act == ACT_GELU) {
            if (p.aux) store_out<OUT>(p.aux, m * p.aux_rs + n, v);
            v = gelu_tanh_f(v);
          }
        }
        store_out<OUT>(p.C, m * p.c_rs + n * p.c_cs, v);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
struct View2D {
  const void* data;
  int64_t rows, cols, rs, cs;
};

View2D view2d(const TensorDesc& t, bool trans) {
  if (!trans) return {t.data, t.shape[0], t.shape[1], t.stride[0], t.stride[1]};
  return {t.data, t.shape[1], t.shape[0], t.stride[1], t.stride[0]};
}

bool stride_valid_2d(const TensorDesc& t) {
  return t.rank == 2 && t.stride[0] > 0 && t.stride[1] > 0;
}

// gemm/launcher.cu:48-70
void read_gemm_attr(const void* attr, bool* ta, bool* tb) {
  *ta = *tb = false;
  const AttrBlob& a = blob(attr);
  if (!attr) return;
  if (a.schema_id != 0 && a.schema_id != AICF_SCHEMA_GEMM) return;
  if (!payload_ok(a, 8)) return;
  *ta = field<int32_t>(a, 0) != 0;
  *tb = field<int32_t>(a, 4) != 0;
}

// Epilogue attributes: GPEL <iii> (transA, transB, relu; relu default 1,
// gemm_epilogue/launcher.cu:57-80) or GEPI <iii> (transA, transB, kind).
struct EpiAttr {
  bool ta = false, tb = false;
  int kind = AICF_EPI_BIAS_RELU;
};
EpiAttr read_epi_attr(const void* attr) {
  EpiAttr e;
  const AttrBlob& a = blob(attr);
  if (!attr) return e;
  if (a.schema_id == AICF_SCHEMA_GEPI) {
    if (!payload_ok(a, 12)) return e;
    e.ta = field<int32_t>(a, 0) != 0;
    e.tb = field<int32_t>(a, 4) != 0;
    e.kind = field<int32_t>(a, 8);
    return e;
  }
  if (a.schema_id != 0 && a.schema_id != AICF_SCHEMA_GPEL) return e;
  if (!payload_ok(a, 12)) return e;
  e.ta = field<int32_t>(a, 0) != 0;
  e.tb = field<int32_t>(a, 4) != 0;
  e.kind = field<int32_t>(a, 8) != 0 ? AICF_EPI_BIAS_RELU : AICF_EPI_BIAS;
  return e;
}

bool epi_kind_valid(int k) { return k >= AICF_EPI_BIAS_RELU && k <= AICF_EPI_DGELU_PARTIALS; }

// gemm/launcher.cu:116-148: A[M,K] . B[K,N] -> C[M,N] with positive strides.
bool gemm_views_ok(const TensorDesc& A0, const TensorDesc& B0, const TensorDesc& C0, bool ta,
                   bool tb) {
  if (A0.rank != 2 || B0.rank != 2 || C0.rank != 2) return false;
  if (!stride_valid_2d(A0) || !stride_valid_2d(B0) || !stride_valid_2d(C0)) return false;
  const View2D A = view2d(A0, ta), B = view2d(B0, tb), C = view2d(C0, false);
  const int64_t M = A.rows, K = A.cols, N = B.cols;
  if (M <= 0 || N <= 0 || K <= 0) return false;
  if (B.rows != K || C.rows != M || C.cols != N) return false;
  if (M > INT32_MAX / 2 || N > INT32_MAX / 2) return false;
  return true;
}

int load_mode(int64_t rs_rows, int64_t cs_k) {
  if (cs_k == 1) return LD_KCONTIG;
  if (rs_rows == 1) return LD_MNCONTIG;
  return LD_GATHER;
}

template <int IN, int OUT, int BM, int BN, int BK, int WM, int WN>
Status run_cfg(GemmParams& p, hipStream_t s) {
  p.tiles_m = (int)((p.M + BM - 1) / BM);
  p.tiles_n = (int)((p.N + BN - 1) / BN);
  const int64_t total = (int64_t)p.tiles_m * p.tiles_n;
  if (total > INT32_MAX) return Status::InvalidArgument;
  gemm_mfma_kernel<IN, OUT, BM, BN, BK, WM, WN><<<(unsigned)total, 64 * WM * WN, 0, s>>>(p);
  return launch_status("gemm_mfma");
}

template <int IN, int OUT, int ACT, int BM, int BN, int WM, int WN, bool AKC, bool BKC, int S = 2>
Status run_nt_act(const GemmParams& g, hipStream_t s) {
  NTParams p{};
  p.A = g.A;
  p.B = g.B;
  p.C = g.C;
  p.bias = g.bias;
  p.aux = g.aux;
  p.lda = AKC ? g.a_rs : g.a_cs;  // memory row stride of A ([M][K] or [K][M])
  p.ldb = BKC ? g.b_cs : g.b_rs;  // memory row stride of B ([N][K] or [K][N])
  p.ldc = g.c_rs;
  p.aux_ld = g.aux_rs;
  p.M = (int)g.M;
  p.N = (int)g.N;
  p.K = (int)g.K;
  p.bias_f32 = g.bias_f32;
  p.tiles_m = (p.M + BM - 1) / BM;
  p.tiles_n = (p.N + BN - 1) / BN;
  p.adam = g.adam;
  p.colsum = g.colsum;
  // 256 x 256 tiles hold one workgroup per CU: with more tiles than CUs, the
  // persistent configuration launches one workgroup per CU (a multiple of 8,
  // one per XCD slot) that loops over its tiles.
  unsigned grid = (unsigned)(p.tiles_m * p.tiles_n);
  if constexpr (nt_persistent(BM, BN, WM, WN)) {
    const int ncu = device_cu_count();
    if (ncu > 0 && ncu % 8 == 0 && grid > (unsigned)ncu) grid = (unsigned)ncu;
  }
  gemm_nt_kernel<IN, OUT, ACT, BM, BN, WM, WN, AKC, BKC, S><<<grid, 64 * WM * WN, 0, s>>>(p);
  return launch_status("gemm_nt");
}

template <int IN, int OUT, int BM, int BN, int WM, int WN, bool AKC, bool BKC, int S = 2>
Status run_nt_layout(const GemmParams& g, hipStream_t s) {
  switch (g.act) {
    case ACT_RELU: return run_nt_act<IN, OUT, ACT_RELU, BM, BN, WM, WN, AKC, BKC, S>(g, s);
    case ACT_GELU: return run_nt_act<IN, OUT, ACT_GELU, BM, BN, WM, WN, AKC, BKC, S>(g, s);
    case ACT_DGELU: return run_nt_act<IN, OUT, ACT_DGELU, BM, BN, WM, WN, AKC, BKC, S>(g, s);
    case ACT_ADAMW:
      if constexpr (IN == IN_BF16 && OUT == OUT_F32)
        return run_nt_act<IN, OUT, ACT_ADAMW, BM, BN, WM, WN, AKC, BKC, S>(g, s);
      return Status::Internal;  // fused AdamW takes bf16 operands and an fp32 gradient
    default: return run_nt_act<IN, OUT, ACT_NONE, BM, BN, WM, WN, AKC, BKC, S>(g, s);
  }
}

// Operand layouts: K-contiguous ([MN][K]) on every tile configuration;
// MN-contiguous ([K][MN], read through the transposing LDS loads for 16-bit
// operands, one 4-byte read per K-row for fp32) where MN_OK (rows of at
// least 16 chunks: 256 x 256 and 128 x 128, and 64 x 64 for fp32).
template <int IN, int OUT, int BM, int BN, int WM, int WN, bool MN_OK, int S = 2>
Status run_nt(const GemmParams& g, hipStream_t s) {
  const bool akc = g.a_mode == LD_KCONTIG, bkc = g.b_mode == LD_KCONTIG;
  if (akc && bkc) return run_nt_layout<IN, OUT, BM, BN, WM, WN, true, true, S>(g, s);
  if constexpr (MN_OK) {
    if (akc) return run_nt_layout<IN, OUT, BM, BN, WM, WN, true, false, S>(g, s);
    if (bkc) return run_nt_layout<IN, OUT, BM, BN, WM, WN, false, true, S>(g, s);
    return run_nt_layout<IN, OUT, BM, BN, WM, WN, false, false, S>(g, s);
  }
  return Status::Internal;  // excluded by nt_eligible
}

// 256 x 256 tiles.  bf16 with K-contiguous operands and a one-output
// epilogue (none, ReLU, GELU): four waves of 128 x 128, one per SIMD, which
// issue the MFMAs back to back.  Everything else: eight waves of 128 x 64; the
// GELU (two outputs) and dGELU (pre-activation read) epilogues move twice
// the bytes per wave with four waves.  f16 keeps eight: four take 4% less on
// several rounds of long K (8192^3 770 us, 740) but 6-9% more at K <= 1024
// (8192 x 4096 x 1024 61.2, 65.1, with GELU 69.6, 75.0).
template <int IN, int OUT>
Status run_nt256(const GemmParams& g, hipStream_t s) {
  if constexpr (IN == IN_BF16) {
    if (g.a_mode == LD_KCONTIG && g.b_mode == LD_KCONTIG) {
      if (g.act == ACT_NONE) return run_nt_act<IN, OUT, ACT_NONE, 256, 256, 2, 2, true, true>(g, s);
      if (g.act == ACT_RELU) return run_nt_act<IN, OUT, ACT_RELU, 256, 256, 2, 2, true, true>(g, s);
      // bias+GELU without the pre-activation output: 8192^3 757 vs 810 us,
      // 8192 x 4096 x 11008 535 vs 559 (same bits); with it the two
      // configurations are equal and the step keeps eight waves
      if (g.act == ACT_GELU && !g.aux)
        return run_nt_act<IN, OUT, ACT_GELU, 256, 256, 2, 2, true, true>(g, s);
    }
  }
  return run_nt<IN, OUT, 256, 256, 2, 4, true>(g, s);
}

// The NT fast path applies to 16-bit and fp32 operands that are each
// K-contiguous ([MN][K]) or, where the caller allows it (mn_ok: the 256 x 256
// and 128 x 128 tiles, and fp32 64 x 64), MN-contiguous ([K][MN]), with 16-byte
// aligned bases and rows; C (and the aux matrix) have unit column stride with
// 16-byte aligned rows, and bias is contiguous.  K is whole K-steps, and the
// shape tiles exactly or, where the output is only written (no update in
// place, no column sums, no operand or pre-activation in the output's memory),
// the last tiles are moved back to end at M and N: columns, and rows of an
// M-contiguous A, then have to be whole 16-byte chunks, and the tiles may hold
// a quarter more than the output (above that the next smaller tile or the edge
// kernel does less work).  bf16 against the edge kernel: 8190 x 4096 x 4096 NT
// 233 -> 184 us, NN 238 -> 190; 1000 x 1000 x 1024 9.5 -> 6.5.
template <int IN, int OUT>
bool nt_eligible(const GemmParams& p, int BM, int BN, bool mn_ok) {
  constexpr int ES = IN == IN_F32 ? 4 : 2;
  auto operand_ok = [&](int mode, int64_t ld_k, int64_t ld_mn, int64_t rows_mn) {
    if (mode == LD_KCONTIG) return (ld_k * ES) % 16 == 0 && rows_mn * ld_k * ES < INT32_MAX;
    if (mode == LD_MNCONTIG && mn_ok) return (ld_mn * ES) % 16 == 0 && p.K * ld_mn * ES < INT32_MAX;
    return false;
  };
  // A view [M, K]: K-contiguous row stride a_rs, MN-contiguous row stride a_cs.
  // B view [K, N]: K-contiguous row stride b_cs, MN-contiguous row stride b_rs.
  if (!operand_ok(p.a_mode, p.a_rs, p.a_cs, BM) || !operand_ok(p.b_mode, p.b_cs, p.b_rs, BN)) return false;
  if (p.K % (128 / ES)) return false;
  if (p.M % BM || p.N % BN) {
    constexpr int64_t CE = 16 / ES, CO = OUT == OUT_F32 ? 4 : 8;
    if (p.act == ACT_ADAMW || p.colsum || !p.apart || p.M < BM || p.N < BN) return false;
    if (p.M % BM && p.a_mode != LD_KCONTIG && p.M % CE) return false;
    if (p.N % BN && (p.N % CO || (p.b_mode != LD_KCONTIG && p.N % CE))) return false;
    if (p.M % 64 == 0 && p.N % 64 == 0) {
      // exact smaller tiles exist: fp32 is bound by its MFMAs and loses by
      // every row computed twice (4160 x 4160 x 512 NN 141 us on 64 x 64, 242
      // here); 16-bit from K = 1024 on, or 768 with one output and a 128 x 128
      // tile a CU (bf16 2048 x 2880 x 1024 NN 29.7 us on 64 x 64, 15.6 here, x 768
      // 17.0, 12.9, but 1600 x 1600 x 768 7.6, 8.4), or 512 with eight of them
      // (5824 x 5824 x 512 76, 46; 6464 x 3136 x 512 with both GELU outputs loses
      // 20%); and 256 x 256 only while they take one round of the CUs (2944 x 2944
      // x 1024 NN 28.6 on 128 x 128, 24.7; 4224 x 4224 x 1024 47.2, 49.4) and,
      // beside 128 x 128 ones, with two outputs or a pre-activation from K = 1536
      // on (8192 x 1152 x 1024 NT with both GELU outputs 30.3, 32.1)
      const int64_t tiles128 = ((p.M + 127) / 128) * ((p.N + 127) / 128);
      const bool one_out = p.act == ACT_NONE || p.act == ACT_RELU || (p.act == ACT_GELU && !p.aux);
      const int64_t from = tiles128 >= 2048 ? 512 : one_out && tiles128 >= 256 ? 768 : 1024;
      if (IN == IN_F32 || p.K < from) return false;
      if (BM == 256 && (((p.M + 255) / 256) * ((p.N + 255) / 256) > 256 ||
                        (!one_out && p.M % 128 == 0 && p.N % 128 == 0 && p.K < 1536)))
        return false;
    }
    const int64_t rows = (p.M + BM - 1) / BM * BM, cols = (p.N + BN - 1) / BN * BN;
    if ((double)rows * cols > 1.25 * (double)p.M * p.N) return false;
    if (p.act == ACT_DGELU) {  // Z read again after a neighbour stored its tile
      const uintptr_t c = (uintptr_t)p.C, z = (uintptr_t)p.aux, osz = OUT == OUT_F32 ? 4 : 2;
      if (c < z + (uintptr_t)(p.M * p.aux_rs) * osz && z < c + (uintptr_t)(p.M * p.c_rs) * osz) return false;
    }
  }
  if ((uintptr_t)p.A % 16 || (uintptr_t)p.B % 16) return false;
  const int osz = OUT == OUT_F32 ? 4 : 2;
  if (p.c_cs != 1 || (uintptr_t)p.C % 16 || (p.c_rs * osz) % 16) return false;
  if (p.aux && (((uintptr_t)p.aux % 16) || (p.aux_rs * osz) % 16)) return false;
  if (p.bias && (p.bias_s != 1 || (uintptr_t)p.bias % 16)) return false;
  if (p.M > INT32_MAX / 2 || p.N > INT32_MAX / 2 || p.K > INT32_MAX / 2) return false;
  return true;
}

// Column sums of a 256 x 256 block of a stored bf16 matrix, row t of
// out [M/256, N] for block row t, in the order of the epilogue's
// copy_out_colsum: a lane takes one 8-column chunk and every 16th row, lanes
// l and l + 32 are added, then the 8 waves in order.
__global__ __launch_bounds__(512) void tile_colsum_kernel(const uint16_t* __restrict__ c, int64_t ldc,
                                                          float* __restrict__ out, int N) {
  __shared__ float red[8][256];
  const int tid = threadIdx.x, n0 = blockIdx.x * 256;
  const uint16_t* src = c + ((int64_t)blockIdx.y * 256 + (tid >> 5)) * ldc + n0 + (tid & 31) * 8;
  u16x8 x[16];
#pragma unroll
  for (int k = 0; k < 16; ++k) x[k] = *reinterpret_cast<const u16x8*>(src + (int64_t)k * 16 * ldc);
  float cs[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) cs[e] = 0.0f;
#pragma unroll
  for (int k = 0; k < 16; ++k)
#pragma unroll
    for (int e = 0; e < 8; ++e) cs[e] += bf16_to_f32(x[k][e]);
#pragma unroll
  for (int e = 0; e < 8; ++e) cs[e] += __shfl_xor(cs[e], 32, 64);
  const int w = tid >> 6, l = tid & 63;
  if (l < 32) {
#pragma unroll
    for (int e = 0; e < 8; ++e) red[w][l * 8 + e] = cs[e];
  }
  __syncthreads();
  if (tid < 256) {
    float s = red[0][tid];
#pragma unroll
    for (int k = 1; k < 8; ++k) s += red[k][tid];
    out[(int64_t)blockIdx.y * N + n0 + tid] = s;
  }
}

template <int IN, int OUT>
Status run_gemm(GemmParams& p, hipStream_t s) {
  p.apart = gemm_outputs_apart(p, IN == IN_F32 ? 4 : 2, OUT == OUT_F32 ? 4 : 2);
  if (p.colsum) {  // dGELU with column sums, bf16 output, M and N multiples of 256
    if constexpr (OUT == OUT_BF16 && IN != IN_F32) {
      if (p.act == ACT_DGELU && nt_eligible<IN, OUT>(p, 256, 256, true)) {
        // the column sums live in the 8-wave 256 x 256 configuration's
        // epilogue (whole tile in one pass): dispatch to it directly
        if ((p.M / 256) * (p.N / 256) >= 128 || !p.apart) return run_nt<IN, OUT, 256, 256, 2, 4, true>(p, s);
        // fewer of those tiles than half the CUs: smaller ones, then the sums
        // from the stored output, in the same order (256 x 3584 x 3584: 72 ->
        // 21 us, 2048^3 49 -> 28; same bits)
        float* colsum = p.colsum;
        p.colsum = nullptr;
        const Status st = run_gemm<IN, OUT>(p, s);
        p.colsum = colsum;
        if (st != Status::Ok) return st;
        tile_colsum_kernel<<<dim3((unsigned)(p.N / 256), (unsigned)(p.M / 256)), 512, 0, s>>>(
            (const uint16_t*)p.C, p.c_rs, colsum, (int)p.N);
        return launch_status("gemm_tile_colsum");
      }
    }
    return Status::NotImplemented;
  }
  if (p.act == ACT_ADAMW) {  // the fused optimizer epilogue: M and N multiples of 256
    if constexpr (OUT == OUT_F32 && IN == IN_BF16) {
      if (nt_eligible<IN, OUT>(p, 256, 256, true)) {
        // the largest tiles that give every other CU one, as for the other
        // epilogues: 1024 x 1024 x 8192 174 -> 37 us, 2048 x 2048 x 8192 181 ->
        // 85, 2560 x 2560 x 4096 122 -> 87 (400 tiles of 128 x 128).  The
        // gradient has the plain product's bits: K order does not depend on the
        // tile, and K is split where the plain product splits it.
        if (edge_splits_k(p, IN)) return edge_gemm(p, IN, OUT, s);
        const int64_t tiles128 = (p.M / 128) * (p.N / 128);
        const bool deep = p.K >= 16 * 64;
        if (tiles128 >= 512 || !p.apart) return run_nt256<IN, OUT>(p, s);
        if (tiles128 >= 128) {
          if (deep && tiles128 <= 256) return run_nt<IN, OUT, 128, 128, 2, 2, true, 4>(p, s);
          return run_nt<IN, OUT, 128, 128, 2, 2, true>(p, s);
        }
        if (deep) return run_nt<IN, OUT, 64, 64, 2, 2, true, 8>(p, s);
        return run_nt<IN, OUT, 64, 64, 2, 2, true>(p, s);
      }
    }
    return Status::NotImplemented;
  }
  if constexpr (IN == IN_F32 && OUT == OUT_F32) {
    // fewer than 128 tiles of 64 x 64: one 16 x 16 tile per wave with K split
    // over the waves of a workgroup reaches more CUs than any tiled
    // configuration, and reads every operand layout in place.  Above 512
    // such tiles (two workgroups a CU) it re-reads the operands from L2 often
    // and long K goes to the edge kernel's K-split tiles: 512 x 512 x 1024 NN
    // 15.8 us, 10.1 there, NT 20.2, 9.4; 300 x 1001 x 2000 NN 45.7, 31.5.  Short
    // K stays, with whole 16 x 16 tiles to K = 511 (512 x 512 x 384 NN 6.5, 8.2;
    // NT 8.0, 8.3), else to 319 (1000 x 200 x 256 NN 5.1, 5.3, NT 6.2, 5.2, x 384
    // 6.6, 6.2; 4096 x 60 x 384 TN 14.4, 6.3), and to 255 from 1408 tiles on (768
    // x 512 x 256 NN 6.7, 6.4, NT 8.0, 6.4).
    const int64_t tiles64 = ((p.M + 63) / 64) * ((p.N + 63) / 64);
    const int64_t tiles16 = ((p.M + 15) / 16) * ((p.N + 15) / 16);
    const bool whole = p.M % 16 == 0 && p.N % 16 == 0 && p.N >= 64;
    const bool split = tiles16 > 512 && p.K >= (tiles16 >= 1408 ? 256 : whole ? 512 : 320) && edge_gemm_ok(p, IN);
    if (tiles64 < kSmallGemmMaxTiles64 && !split && (p.act == ACT_NONE || p.act == ACT_RELU) && p.c_cs == 1 && !p.aux) {
      SmallGemm g{};
      g.A = (const float*)p.A;
      g.B = (const float*)p.B;
      g.C = (float*)p.C;
      g.bias = (const float*)p.bias;
      g.a_m = p.a_rs;
      g.a_k = p.a_cs;
      g.b_k = p.b_rs;
      g.b_n = p.b_cs;
      g.c_m = p.c_rs;
      g.bias_s = p.bias_s;
      g.M = p.M;
      g.N = p.N;
      g.K = p.K;
      g.relu = p.act == ACT_RELU;
      if (small_gemm_ok(g)) return small_gemm_f32(g, s);
    }
    // at most half a 64 x 64 tile a CU: K split over groups of waves (512 x
    // 1024 x 4096 67 -> 46 us, 1856 x 184 x 3392 TN 54 -> 40)
    const int64_t tiles64x32 = ((p.M + 63) / 64) * ((p.N + 31) / 32);
    if (tiles64x32 <= 256 && p.K >= 512 && edge_gemm_ok(p, IN)) return edge_gemm(p, IN, OUT, s);
  }
  {
    constexpr bool MN = true;
    const int64_t tiles256 = ((p.M + 255) / 256) * ((p.N + 255) / 256);
    const int64_t tiles128 = ((p.M + 127) / 128) * ((p.N + 127) / 128);
    // K <= 512 (at most 8 K-steps) with a one-output epilogue (none, bias,
    // ReLU): a 256 x 256 tile's loads and stores are no longer covered by its
    // MFMA work, and 128 x 128 tiles, two workgroups per CU, overlap one
    // tile's epilogue with another's K loop (8192 x 4096 x 256: 30.5 vs 36
    // us, x 512: 42.7 vs 46).  16-bit bias+GELU without the pre-activation
    // output too at K <= 256 (x 256: 33.4 vs 36.5 us on the 8-wave 256 x 256
    // tiles); at K = 512 GELU stays on 256 x 256 (45 vs 48-50 us).
    // K-contiguous operands only; the others keep 256.
    const bool one_out = p.act == ACT_NONE || p.act == ACT_RELU ||
                         (IN != IN_F32 && p.act == ACT_GELU && !p.aux && p.K <= 256);
    if (p.K <= 512 && one_out && tiles128 >= 256 && (p.K <= 256 || IN == IN_F32) &&
        nt_eligible<IN, OUT>(p, 128, 128, false)) {
      // 16-bit: 8 waves of 64 x 32 (8192 x 4096 x 256: 28.3 vs 29.4-31.3 us
      // none, 33.7 vs 35.2-36.0 GELU against 4 waves of 64 x 64)
      if constexpr (IN != IN_F32) return run_nt<IN, OUT, 128, 128, 2, 4, false>(p, s);
      return run_nt<IN, OUT, 128, 128, 2, 2, false>(p, s);
    }
    // Other 16-bit GEMMs with K <= 512 and at least one 256 x 256 tile per
    // CU: the 8-wave persistent tiles (8192 x 4096 x 512: 41.4 vs 46.0 us
    // none, 48.0 vs 52.5 GELU; x 256 with GELU: 38.4 vs 42.2 us against the
    // 4-wave 256 x 256 tiles, same bits).
    if constexpr (IN != IN_F32) {
      if (p.K <= 512 && tiles256 >= 256 && nt_eligible<IN, OUT>(p, 256, 256, MN))
        return run_nt<IN, OUT, 256, 256, 2, 4, MN>(p, s);
    }
    if (tiles256 >= 128 && nt_eligible<IN, OUT>(p, 256, 256, MN)) return run_nt256<IN, OUT>(p, s);
    // 16-bit operands with at least 16 K-steps: small tiles take deeper
    // pipelines (a K-step is a few hundred cycles of MFMA work per wave, less
    // than a load's latency).  128 x 128 with 4 stages needs all of LDS, so
    // only where one workgroup per CU is all the grid gives anyway.
    const bool deep = IN != IN_F32 && p.K >= 16 * (128 / (IN == IN_F32 ? 4 : 2));
    // 128 x 128 and 64 x 64 tiles read every operand layout (2048^3 bf16 NN
    // 112.6 -> 19.8 us, fp32 1024^3 NN 53.8 -> 19.7 us against the
    // general-stride kernel)
    constexpr bool MN64 = true;
    // fp32 is bound by its MFMAs, so by the work of the fullest CU, counted here
    // in 64 x 64 tiles: 2048 x 1024 x 512 takes 33.5 us as one 128 x 128 tile on
    // each of 128 CUs, 17.9 as two 64 x 64 tiles each; 2048 x 2176 x 2048 233,
    // 151.  Where both load it alike, short K gains from the finer tiles (2048 x
    // 1792 x 128 12.1, 11.0), long K from reading half the operand bytes (2048 x
    // 2048 x 4096 NT 236, 254).  From 384 tiles of 128 x 128 on, 128 x 128.
    const int64_t round64 = (((p.M + 63) / 64) * ((p.N + 63) / 64) + 255) / 256, round128 = 4 * ((tiles128 + 255) / 256);
    const bool smaller = IN == IN_F32 && p.apart && tiles128 < 384 &&
                         (round64 < round128 || (round64 == round128 && p.K <= 512));
    if (tiles128 >= 128 && !smaller && nt_eligible<IN, OUT>(p, 128, 128, true)) {
      if constexpr (IN != IN_F32) {
        if (deep && tiles128 <= 256) return run_nt<IN, OUT, 128, 128, 2, 2, true, 4>(p, s);
      }
      return run_nt<IN, OUT, 128, 128, 2, 2, true>(p, s);
    }
    if constexpr (IN != IN_F32) {
      if (edge_splits_k(p, IN)) return edge_gemm(p, IN, OUT, s);
    }
    // fewer tiles than CUs at 128x128: 64x64 tiles (4 waves of 32x32)
    if (nt_eligible<IN, OUT>(p, 64, 64, MN64)) {
      if constexpr (IN != IN_F32) {
        if (deep) return run_nt<IN, OUT, 64, 64, 2, 2, MN64, 8>(p, s);
      }
      return run_nt<IN, OUT, 64, 64, 2, 2, MN64>(p, s);
    }
    if (nt_eligible<IN, OUT>(p, 128, 128, true)) {
      if constexpr (IN != IN_F32) {
        if (deep) return run_nt<IN, OUT, 128, 128, 2, 2, true, 4>(p, s);
      }
      return run_nt<IN, OUT, 128, 128, 2, 2, true>(p, s);
    }
  }
  // shapes no tile divides, unaligned rows
  if (edge_gemm_ok(p, IN)) return edge_gemm(p, IN, OUT, s);
  // What is left: strides with no contiguous dimension, a strided output, K
  // or a contiguous extent of less than 16 bytes.  Large problems: 128x128
  // workgroup tiles (4 waves, 64x64 per wave).  Smaller ones: 64x64 tiles so
  // that enough workgroups exist.
  const int64_t big_tiles = ((p.M + 127) / 128) * ((p.N + 127) / 128);
  if (big_tiles >= 512) return run_cfg<IN, OUT, 128, 128, (IN == IN_F32 ? 32 : 64), 2, 2>(p, s);
  return run_cfg<IN, OUT, 64, 64, (IN == IN_F32 ? 32 : 64), 2, 2>(p, s);
}

int in_kind(DType d) {
  return d == DType::kF32 ? IN_F32 : d == DType::kF16 ? IN_F16 : IN_BF16;
}

Status dispatch_gemm(GemmParams& p, DType din, DType dout, hipStream_t s) {
  const int ik = in_kind(din);
  if (ik == IN_F32 && dout == DType::kF32) return run_gemm<IN_F32, OUT_F32>(p, s);
  if (ik == IN_F16 && dout == DType::kF16) return run_gemm<IN_F16, OUT_F16>(p, s);
  if (ik == IN_F16 && dout == DType::kF32) return run_gemm<IN_F16, OUT_F32>(p, s);
  if (ik == IN_BF16 && dout == DType::kBF16) return run_gemm<IN_BF16, OUT_BF16>(p, s);
  if (ik == IN_BF16 && dout == DType::kF32) return run_gemm<IN_BF16, OUT_F32>(p, s);
  return Status::InvalidArgument;
}

void fill_operands(GemmParams& p, const TensorDesc& A0, const TensorDesc& B0, const TensorDesc& C0,
                   bool ta, bool tb) {
  const View2D A = view2d(A0, ta), B = view2d(B0, tb), C = view2d(C0, false);
  p.A = A.data;
  p.B = B.data;
  p.C = const_cast<void*>(C.data);
  p.M = A.rows;
  p.K = A.cols;
  p.N = B.cols;
  p.a_rs = A.rs;
  p.a_cs = A.cs;
  p.b_rs = B.rs;
  p.b_cs = B.cs;
  p.c_rs = C.rs;
  p.c_cs = C.cs;
  p.a_mode = load_mode(A.rs, A.cs);
  p.b_mode = load_mode(B.cs, B.rs);  // B tile rows are N, K stride is b_rs
  p.bias = nullptr;
  p.aux = nullptr;
  p.act = ACT_NONE;
}

// ---- Gemm variants --------------------------------------------------------
bool gemm_check(const TensorDesc* in, int ni, const TensorDesc* out, int no, const void* attr,
                DType din, DType dout, bool c_rowmajor) {
  if (!in || !out || ni != 2 || no != 1) return false;
  if (dt(in[0]) != din || dt(in[1]) != din || dt(out[0]) != dout) return false;
  bool ta, tb;
  read_gemm_attr(attr, &ta, &tb);
  if (!gemm_views_ok(in[0], in[1], out[0], ta, tb)) return false;
  return !c_rowmajor || is_contig_2d_rowmajor(out[0]);
}

Status gemm_launch_common(const TensorDesc* in, TensorDesc* out, const void* attr, DType din,
                          DType dout, void* stream) {
  bool ta, tb;
  read_gemm_attr(attr, &ta, &tb);
  GemmParams p{};
  fill_operands(p, in[0], in[1], out[0], ta, tb);
  return dispatch_gemm(p, din, dout, as_stream(stream));
}

#define GEMM_VARIANT(NAME, DIN, DOUT, CROW)                                                       \
  bool NAME##_sup(const TensorDesc* i, int ni, const TensorDesc* o, int no, const void* a) {     \
    return gemm_check(i, ni, o, no, a, DIN, DOUT, CROW);                                          \
  }                                                                                               \
  Status NAME##_launch(const TensorDesc* i, int ni, TensorDesc* o, int no, const void* a, void*, \
                       size_t, void* s) {                                                         \
    if (!NAME##_sup(i, ni, o, no, a)) return Status::InvalidArgument;                            \
    return gemm_launch_common(i, o, a, DIN, DOUT, s);                                             \
  }

GEMM_VARIANT(gemm_f32, DType::kF32, DType::kF32, false)
GEMM_VARIANT(gemm_f16, DType::kF16, DType::kF16, true)
GEMM_VARIANT(gemm_bf16, DType::kBF16, DType::kBF16, false)
GEMM_VARIANT(gemm_bf16_f32out, DType::kBF16, DType::kF32, false)

// ---- GemmEpilogue variants ------------------------------------------------
// inputs (A, B, X): X is the bias [N] (kinds 0..4) or Z [M,N] (kind 5).
// outputs (C) or (C, Zaux) for BIAS_GELU.
bool epi_check(const TensorDesc* in, int ni, const TensorDesc* out, int no, const void* attr,
               DType din, DType dout, bool c_rowmajor) {
  if (!in || !out || ni != 3 || no < 1 || no > 3) return false;
  if (dt(in[0]) != din || dt(in[1]) != din || dt(out[0]) != dout) return false;
  const EpiAttr e = read_epi_attr(attr);
  if (!epi_kind_valid(e.kind)) return false;
  if (!gemm_views_ok(in[0], in[1], out[0], e.ta, e.tb)) return false;
  if (c_rowmajor && !is_contig_2d_rowmajor(out[0])) return false;
  const View2D C = view2d(out[0], false);
  const TensorDesc& X = in[2];
  if (e.kind == AICF_EPI_DGELU_COLSUM || e.kind == AICF_EPI_DGELU_PARTIALS) {
    // outputs (C, db [N] f32, workspace [P >= M/256, N] f32), or (C,
    // partials [P >= M/256, N] f32); bf16 output
    const bool fin = e.kind == AICF_EPI_DGELU_COLSUM;
    if (no != (fin ? 3 : 2) || dout != DType::kBF16 || !is_contig_2d_rowmajor(out[0])) return false;
    if (dt(X) != dout || X.rank != 2 || X.shape[0] != C.rows || X.shape[1] != C.cols) return false;
    if (X.stride[1] != 1 || X.stride[0] <= 0) return false;
    const TensorDesc &D = out[1], &W = out[fin ? 2 : 1];
    if (fin && (dt(D) != DType::kF32 || !D.contiguous || D.rank != 1 || D.shape[0] != C.cols)) return false;
    if (dt(W) != DType::kF32 || !W.contiguous || W.rank != 2 || W.shape[1] != C.cols ||
        W.shape[0] < C.rows / 256)
      return false;
    if (!fin && W.shape[0] != C.rows / 256) return false;  // its reader sums every row
    // the column sums are kept per 256-row block: accept exactly the shapes
    // that run_gemm takes with them (M, N multiples of 256, so the workspace
    // has at least one row; K of 64; aligned operands), also of a descriptor
    // whose workspace has no memory yet
    if (din != DType::kBF16 || C.rows % 256 || C.cols % 256) return false;
    GemmParams p{};
    fill_operands(p, in[0], in[1], out[0], e.ta, e.tb);
    p.act = ACT_DGELU;
    p.aux = const_cast<void*>(X.data);
    p.aux_rs = X.stride[0];
    return nt_eligible<IN_BF16, OUT_BF16>(p, 256, 256, true);
  }
  if (no > 2) return false;
  if (e.kind == AICF_EPI_DGELU) {
    if (no != 1) return false;
    if (dt(X) != dout || X.rank != 2 || X.shape[0] != C.rows || X.shape[1] != C.cols) return false;
    if (X.stride[1] != 1 || X.stride[0] <= 0) return false;
  } else {
    // bias: rank 1, length N, positive stride; dtype = input dtype, or fp32
    if (X.rank != 1 || X.stride[0] <= 0 || X.shape[0] != C.cols) return false;
    if (dt(X) != din && dt(X) != DType::kF32) return false;
    if (dt(X) != dout && dt(X) != DType::kF32) return false;
  }
  if (no == 2) {
    if (e.kind != AICF_EPI_BIAS_GELU) return false;
    const TensorDesc& Z = out[1];
    if (dt(Z) != dout || Z.rank != 2 || Z.shape[0] != C.rows || Z.shape[1] != C.cols) return false;
    if (Z.stride[1] != 1 || Z.stride[0] <= 0) return false;
  }
  return true;
}

Status epi_launch_common(const TensorDesc* in, int no, TensorDesc* out, const void* attr, DType din,
                         DType dout, void* stream) {
  const EpiAttr e = read_epi_attr(attr);
  GemmParams p{};
  fill_operands(p, in[0], in[1], out[0], e.ta, e.tb);
  const TensorDesc& X = in[2];
  switch (e.kind) {
    case AICF_EPI_BIAS_RELU: p.act = ACT_RELU; break;
    case AICF_EPI_BIAS: p.act = ACT_NONE; break;
    case AICF_EPI_RELU: p.act = ACT_RELU; break;
    case AICF_EPI_BIAS_GELU: p.act = ACT_GELU; break;
    case AICF_EPI_GELU: p.act = ACT_GELU; break;
    case AICF_EPI_DGELU: p.act = ACT_DGELU; break;
    case AICF_EPI_DGELU_COLSUM: p.act = ACT_DGELU; break;
    case AICF_EPI_DGELU_PARTIALS: p.act = ACT_DGELU; break;
  }
  const bool with_bias = e.kind == AICF_EPI_BIAS_RELU || e.kind == AICF_EPI_BIAS ||
                         e.kind == AICF_EPI_BIAS_GELU;
  if (with_bias) {
    p.bias = X.data;
    p.bias_s = X.stride[0];
    p.bias_f32 = dt(X) == DType::kF32 ? 1 : 0;
  }
  if (e.kind == AICF_EPI_DGELU || e.kind == AICF_EPI_DGELU_COLSUM || e.kind == AICF_EPI_DGELU_PARTIALS) {
    p.aux = const_cast<void*>(X.data);
    p.aux_rs = X.stride[0];
  } else if (no == 2) {
    p.aux = out[1].data;
    p.aux_rs = out[1].stride[0];
  }
  if (e.kind == AICF_EPI_DGELU_PARTIALS) {  // the column sums are finished by a later op
    p.colsum = (float*)out[1].data;
    return dispatch_gemm(p, din, dout, as_stream(stream));
  }
  if (e.kind == AICF_EPI_DGELU_COLSUM) {
    if (!out[2].data) return Status::InvalidArgument;
    p.colsum = (float*)out[2].data;
    const Status st = dispatch_gemm(p, din, dout, as_stream(stream));
    if (st != Status::Ok) return st;
    return colsum_finish(p.colsum, (float*)out[1].data, p.M / 256, p.N, stream);
  }
  return dispatch_gemm(p, din, dout, as_stream(stream));
}

#define EPI_VARIANT(NAME, DIN, DOUT, CROW)                                                        \
  bool NAME##_sup(const TensorDesc* i, int ni, const TensorDesc* o, int no, const void* a) {     \
    return epi_check(i, ni, o, no, a, DIN, DOUT, CROW);                                           \
  }                                                                                               \
  Status NAME##_launch(const TensorDesc* i, int ni, TensorDesc* o, int no, const void* a, void*, \
                       size_t, void* s) {                                                         \
    if (!NAME##_sup(i, ni, o, no, a)) return Status::InvalidArgument;                            \
    return epi_launch_common(i, no, o, a, DIN, DOUT, s);                                          \
  }

EPI_VARIANT(epi_f32, DType::kF32, DType::kF32, false)
EPI_VARIANT(epi_f16, DType::kF16, DType::kF16, true)
EPI_VARIANT(epi_bf16, DType::kBF16, DType::kBF16, false)
EPI_VARIANT(epi_bf16_f32out, DType::kBF16, DType::kF32, false)

// ---------------------------------------------------------------------------
// GemmAdamW (no reference counterpart): the weight-gradient GEMM of a Linear
// layer with AdamW applied in its epilogue, so the fp32 gradient never goes
// to memory.  inputs (A bf16, B bf16, P f32, M f32, V f32, step i32 scalar),
// outputs (P, M, V in place, Wb bf16 shadow of P); P, M, V, Wb are [M, N]
// row-major views; grad = op(A) . op(B).  Attr schema GADW
// <ii fffff>: transA, transB, lr, beta1, beta2, eps, weight_decay.  M and N
// multiples of 256, K of 64, 16-byte aligned rows; other shapes are not
// supported.
// ---------------------------------------------------------------------------
struct GadwAttr {
  bool ta = false, tb = false;
  AdamWArgs args{};
  bool ok = false;
};
GadwAttr read_gadw(const void* attr) {
  GadwAttr g;
  const AttrBlob& a = blob(attr);
  if (!attr || a.schema_id != AICF_SCHEMA_GADW || !payload_ok(a, 28)) return g;
  g.ta = field<int32_t>(a, 0) != 0;
  g.tb = field<int32_t>(a, 4) != 0;
  const float lr = field<float>(a, 8), b1 = field<float>(a, 12), b2 = field<float>(a, 16);
  const float eps = field<float>(a, 20), wd = field<float>(a, 24);
  if (lr != lr || b1 != b1 || b2 != b2 || eps != eps || wd != wd) return g;
  g.args = AdamWArgs{lr, b1, b2, eps, wd, 1.0f - b1, 1.0f - b2, 1.0f - lr * wd};
  g.ok = true;
  return g;
}

bool gadw_fill(const TensorDesc* in, int ni, const TensorDesc* out, int no, const void* attr,
               GemmParams* pp) {
  if (!in || !out || ni != 6 || no != 4) return false;
  const GadwAttr at = read_gadw(attr);
  if (!at.ok) return false;
  if (dt(in[0]) != DType::kBF16 || dt(in[1]) != DType::kBF16) return false;
  for (int k = 2; k < 5; ++k)
    if (dt(in[k]) != DType::kF32 || !is_contig_2d_rowmajor(in[k])) return false;
  if (dt(in[5]) != DType::kI32 || !in[5].contiguous || numel_of(in[5]) != 1) return false;
  for (int k = 0; k < 3; ++k)  // P, M, V updated in place
    if (dt(out[k]) != DType::kF32 || out[k].data != in[k + 2].data || !same_shape(out[k], in[k + 2]))
      return false;
  if (dt(out[3]) != DType::kBF16 || !is_contig_2d_rowmajor(out[3]) || !same_shape(out[3], in[2])) return false;
  if (!same_shape(in[2], in[3]) || !same_shape(in[2], in[4])) return false;
  if (!gemm_views_ok(in[0], in[1], in[2], at.ta, at.tb)) return false;
  GemmParams p{};
  fill_operands(p, in[0], in[1], in[2], at.ta, at.tb);
  p.act = ACT_ADAMW;
  p.adam = GemmAdamW{(float*)in[2].data, (float*)in[3].data, (float*)in[4].data, (uint16_t*)out[3].data,
                     (const int32_t*)in[5].data, at.args};
  if ((uintptr_t)p.adam.M % 16 || (uintptr_t)p.adam.V % 16 || (uintptr_t)p.adam.Wb % 8) return false;
  if (!nt_eligible<IN_BF16, OUT_F32>(p, 256, 256, true)) return false;
  if (pp) *pp = p;
  return true;
}
bool gadw_sup(const TensorDesc* i, int ni, const TensorDesc* o, int no, const void* a) {
  return gadw_fill(i, ni, o, no, a, nullptr);
}
Status gadw_launch(const TensorDesc* i, int ni, TensorDesc* o, int no, const void* a, void*, size_t,
                   void* s) {
  GemmParams p{};
  if (!gadw_fill(i, ni, o, no, a, &p)) return Status::InvalidArgument;
  return run_gemm<IN_BF16, OUT_F32>(p, as_stream(s));
}

size_t no_workspace(const TensorDesc*, int, const void*) { return 0; }

KernelVariant make(const char* name, LaunchFn l, SupportedFn s) {
  KernelVariant v;
  v.name = name;
  v.launch = l;
  v.supported = s;
  v.query_workspace = no_workspace;
  return v;
}

}  // namespace

KernelVariant make_gemm_f32_naive_variant() {
  return make("gemm_f32_mfma", gemm_f32_launch, gemm_f32_sup);
}
KernelVariant make_gemm_f16_tc_wmma_out_f16_variant() {
  return make("gemm_f16_mfma", gemm_f16_launch, gemm_f16_sup);
}
KernelVariant make_gemm_bf16_variant() {
  return make("gemm_bf16_mfma", gemm_bf16_launch, gemm_bf16_sup);
}
KernelVariant make_gemm_bf16_f32out_variant() {
  return make("gemm_bf16_mfma_f32out", gemm_bf16_f32out_launch, gemm_bf16_f32out_sup);
}
KernelVariant make_gemm_bias_relu_f32_naive_variant() {
  return make("gemm_epilogue_f32_mfma", epi_f32_launch, epi_f32_sup);
}
KernelVariant make_gemm_bias_relu_f16_tc_wmma_out_f16_variant() {
  return make("gemm_epilogue_f16_mfma", epi_f16_launch, epi_f16_sup);
}
KernelVariant make_gemm_epilogue_bf16_variant() {
  return make("gemm_epilogue_bf16_mfma", epi_bf16_launch, epi_bf16_sup);
}
KernelVariant make_gemm_epilogue_bf16_f32out_variant() {
  return make("gemm_epilogue_bf16_mfma_f32out", epi_bf16_f32out_launch, epi_bf16_f32out_sup);
}
KernelVariant make_gemm_adamw_bf16_variant() {
  KernelVariant v = make("gemm_adamw_bf16_mfma", gadw_launch, gadw_sup);
  v.expected_attr_schema_id = AICF_SCHEMA_GADW;
  return v;
}

}  // namespace aicf::hip
