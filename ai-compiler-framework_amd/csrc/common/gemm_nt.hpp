// The tiled MFMA GEMM of gfx950, shared by the GEMM ops (gemm.hip) and the ops
// that add epilogues of their own to it (linear_xent.hip).
#pragma once

#include <type_traits>
#include <utility>

#include "gemm_types.hpp"
#include "lds_load.hpp"
#include "linear_xent_plan.hpp"

namespace aicf::hip {

namespace {

// ---------------------------------------------------------------------------
// Tiled MFMA path for tile-divisible shapes: 16-bit operands (each
// K-contiguous or M/N-contiguous) and fp32 operands (K-contiguous).
//   * BM x BN workgroup tiles; a stage holds 128 bytes of K per row (64
//     16-bit or 32 fp32 elements); WM x WN waves (one or two per SIMD for
//     the 256x256 tile), each owning (BM/WM) x (BN/WN) = TM x TN blocks of
//     32x32 fp32 accumulators (v_mfma_f32_32x32x16_bf16/f16, or 4 x
//     v_mfma_f32_32x32x2f32 per 16-byte fp32 fragment);
//   * global -> LDS with gfx950's direct 16-byte LDS loads
//     (buffer_load_dwordx4 ... lds): lane i of a wave fills bytes
//     [16i, 16i+16) of a 1 KB LDS block, so there is no VGPR staging and no
//     ds_write; the XOR swizzle that keeps the fragment reads bank-conflict
//     free is applied by choosing which global chunk each lane fetches;
//   * two LDS stages and one barrier per K-step, placed before the last
//     sub-step so that no wave waits on LDS after it;
//   * the MFMA fragments of sub-step s+1 are read from LDS while the MFMAs of
//     sub-step s run (two register sets), spread over the MFMAs
//     (sched_group_barrier); with K-contiguous operands the next K-step's
//     loads are spread over two sub-steps as well (all at once, they back up
//     the address queue of the CU and stall the MFMA issue);
//   * MFMA operands swapped (A-operand = W rows, B-operand = X rows) so that
//     each lane holds 4 consecutive output columns of one row;
//   * the epilogue stages the output tile through LDS and stores whole rows;
//   * the activation is a template parameter; bias and the pre-activation
//     output are uniform runtime flags.
// ---------------------------------------------------------------------------
typedef __attribute__((address_space(3))) void lds_void_t;
typedef __attribute__((address_space(1))) void glb_void_t;

// What the linear cross-entropy's products carry beside the operands (ACT_LX_*
// only, linear_xent.hip).  Their number of rows is known on the device alone,
// and their last tiles run over the edges of M, N and K: loads past an operand
// return zero, stores are checked.
struct LxArgs {
  const int32_t* n;      // rows that count: M, or K with rows_are_k
  int rows_are_k;
  int a_mn, b_mn;        // extents of A's and B's rows (M/N-contiguous: columns) in memory
  // dX: K is divided into shares (chosen on the device: how many rows count is
  // known there alone).  ACT_LX_SLAB: share s writes slab s of C; the only one,
  // with `direct`, writes `direct` itself as ACT_LX_OUT does C.
  const int32_t* shares;
  void* direct;
  int64_t ld_direct;
  int k_piece;           // K that the shares divide
  int k_before;          // K of the piece whose sums the slabs hold (0: none), to be added to
  // ACT_LX_STATS, ACT_LX_GRAD: logits
  int v0;                // class of column 0
  const int32_t* label;  // class of each row
  float* zlab;           // logit of that class
  float2* stats;         // [tiles_n][stats_ld]: maximum and sum over a tile's classes
  int64_t stats_ld;
  int keep_from;         // columns from here on go to C as exp(z - tile maximum)
  const float* row_max;  // ACT_LX_GRAD: C = exp(z - row_max) row_f, row_g at the label
  const float* row_f;
  const float* row_g;
  // ACT_LX_OUT: C[row_map ? row_map[m] : m] = acc * *alpha
  const float* alpha;
  const int32_t* row_map;
  int vec;               // C's rows lie on 16-byte steps (a slab's always do)
  int add;               // (ACT_LX_SLAB, set by the kernel: this share's slab holds sums)
};

struct NTParams {
  const void* A;      // K-contiguous [M, K] or M-contiguous [K, M], row stride lda (elements)
  const void* B;      // K-contiguous [N, K] or N-contiguous [K, N], row stride ldb (elements)
  void* C;            // [M, N], row stride ldc
  const void* bias;
  void* aux;
  int64_t lda, ldb, ldc, aux_ld;
  int M, N, K;
  int bias_f32;
  int tiles_m, tiles_n;
  GemmAdamW adam;  // ACT_ADAMW only
  float* colsum;   // see GemmParams::colsum
  LxArgs lx;       // ACT_LX_* only
};

// Epilogue of the NT kernels.  Block (i, j) of the accumulators holds D[n][m]
// (MS x MS, see col_of below for the lane's elements).  The fragments go
// through LDS (`smem`, at least
// STAGE_BYTES, free when this is called) so that every global store, and the
// load of the dGELU pre-activation, moves whole 512-1024 byte rows.  LDS rows
// hold 16-byte chunks XOR-swizzled by row, which keeps both the fragment
// writes (32 rows, one chunk each) and the row reads bank-balanced.  A tile
// that does not fit (fp32 256x256) is done in passes over the wave's MS-row
// fragment groups.
template <int MS>
using nt_acc_t = typename std::conditional<MS == 16, floatx4, floatx16>::type;

template <int OUT, int ACT, int BM, int BN, int WM, int WN, int STAGE_BYTES, int MS>
__device__ __forceinline__ void nt_epilogue_staged(const NTParams& p,
                                                   nt_acc_t<MS> (&acc)[BN / WN / MS][BM / WM / MS],
                                                   uint8_t* smem, int m0, int n0) {
  constexpr int NW = WM * WN;
  constexpr int WTM = BM / WM, WTN = BN / WN;
  constexpr int TM = WTM / MS, TN = WTN / MS;
  // 32 x 32 blocks: lane (fr, fh) holds row fr, columns 8 g + 4 fh + {0..3}
  // in acc[..][4 g .. 4 g + 3] (g = 0..3); 16 x 16 blocks: row fr, columns
  // 4 fh + {0..3} in acc[0..3].
  constexpr int G = MS == 32 ? 4 : 1;
  // The lane's coordinates come from a thread index the compiler cannot see
  // through (see opaque_tid below): the LDS slots derived from them are then
  // computed here rather than hoisted out of the persistent tile loop and
  // spilled across the K loop.
  int tid_e = threadIdx.x;
  asm volatile("" : "+v"(tid_e));
  const int lane = tid_e & 63, wave = tid_e >> 6;
  const int wm = wave / WN, wn = wave % WN;
  const int fr = lane % MS, fh = lane / MS;
  auto col_of = [&](int i, int g) -> int { return wn * WTN + i * MS + (MS == 32 ? 8 * g + 4 * fh : 4 * fh); };
  constexpr int NT = 64 * NW;
  constexpr int OB = OUT == OUT_F32 ? 4 : 2;
  // Output stores with the nontemporal hint (no L2 allocation), except on
  // the persistent 8-wave 256 x 256 tiles.  Elsewhere workgroups reach their
  // epilogues at different times, and 128-256 KB of cached output per CU
  // evicts the operand panels the other workgroups of the XCD are still
  // streaming (8192 x 4096 x 11008: 506 -> 469 us, x 256: 24.9 -> 23.0 us,
  // 8192^3: 702 -> 688 us).  The persistent tiles finish their K loops
  // together, and there the train step's next GEMM finds the cached output
  // (its step ran 1.2% slower with nontemporal stores).
  constexpr bool NT_STORE = !(BM == 256 && BN == 256 && NW == 8);
  auto store16 = [&](void* dst, const u16x8& x) {
    if constexpr (NT_STORE)
      __builtin_nontemporal_store(x, reinterpret_cast<u16x8*>(dst));
    else
      *reinterpret_cast<u16x8*>(dst) = x;
  };
  constexpr int ROWB = BN * OB;    // bytes per staged row
  constexpr int CPR = ROWB / 16;   // 16-byte chunks per row
  // GELU stages the pre-activation z and the activation side by side (two
  // regions of half the staging bytes, so half the rows per pass): the
  // accumulators of a pass are dead once both are staged, and none are live
  // beside the copies of the other outputs.
  constexpr bool GELU_DUAL = ACT == ACT_GELU;
  constexpr int REGION = GELU_DUAL ? STAGE_BYTES / 2 : STAGE_BYTES;
  constexpr int ROWS_PASS = REGION / ROWB < BM ? REGION / ROWB : BM;
  constexpr int NPASS = BM / ROWS_PASS;
  constexpr int JP = TM / NPASS;   // MS-row fragment groups per wave per pass
  constexpr int WROWS = JP * MS;   // rows per wave per pass
  static_assert(NPASS * ROWS_PASS == BM && JP * NPASS == TM, "pass split");
  static_assert((CPR & (CPR - 1)) == 0 && (ROWS_PASS * CPR) % NT == 0, "chunk split");
  uint8_t* const tile = smem;

  // Bias of the lane's columns.  32 x 32 blocks: added to the accumulators
  // in place (8 floats per block).  16 x 16 blocks: the lane's 4 x TN bias
  // values are loaded once and added where each fragment is staged; an
  // in-place pass over 32 small accumulator blocks behind the runtime bias
  // test makes the compiler materialise all of them a second time and spill.
  constexpr bool HAS_BIAS_ACT = ACT != ACT_DGELU && ACT != ACT_ADAMW;
  const bool with_bias = HAS_BIAS_ACT && p.bias != nullptr;
  auto bias4 = [&](int i, int g, float* b) {
    const int n = n0 + col_of(i, g);
    if (p.bias_f32) {
      const f32x4 bv = *reinterpret_cast<const f32x4*>((const float*)p.bias + n);
#pragma unroll
      for (int e = 0; e < 4; ++e) b[e] = bv[e];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) b[e] = load_out<OUT>(p.bias, n + e);
    }
  };
  constexpr int BI = MS == 16 ? TN : 1;
  float bias_v[BI][4];
#pragma unroll
  for (int i = 0; i < BI; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) bias_v[i][e] = 0.0f;
  if constexpr (HAS_BIAS_ACT) {
    if (with_bias) {
      if constexpr (MS == 16) {
#pragma unroll
        for (int i = 0; i < TN; ++i) bias4(i, 0, bias_v[i]);
      } else {
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
          for (int g = 0; g < G; ++g) {
            float b[4];
            bias4(i, g, b);
#pragma unroll
            for (int j = 0; j < TM; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[i][j][4 * g + e] += b[e];
          }
      }
    }
  }
  // accumulators of fragment (j, i, g), plus the bias for 16 x 16 blocks
  auto frag4 = [&](int j, int i, int g, float* v) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = acc[i][j][4 * g + e];
    if constexpr (MS == 16) {
      if (with_bias) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += bias_v[i][e];
      }
    }
  };

  // byte offset of this lane's 4 outputs of fragment (jj, i, g) in the tile
  auto slot = [&](int jj, int i, int g) -> int {
    const int pr = wm * WROWS + jj * MS + fr;
    const int cb = col_of(i, g) * OB;  // byte of the 4 outputs in the row
    const int c = cb / 16, half = cb % 16;
    return pr * ROWB + ((c ^ (pr & (CPR - 1))) * 16) + half;
  };
  auto put4 = [&](int off, const float* v) {
    if constexpr (OB == 4) {
      *reinterpret_cast<f32x4*>(tile + off) = f32x4{v[0], v[1], v[2], v[3]};
    } else if constexpr (OUT == OUT_BF16) {
      typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
      *reinterpret_cast<u32x2*>(tile + off) = u32x2{f32x2_to_bf16x2(v[0], v[1]), f32x2_to_bf16x2(v[2], v[3])};
    } else {
      u16x4 o;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = f32_to_f16(v[e]);
      *reinterpret_cast<u16x4*>(tile + off) = o;
    }
  };
  auto get4 = [&](int off, float* v) {
    if constexpr (OB == 4) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(tile + off);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = x[e];
    } else {
      const u16x4 x = *reinterpret_cast<const u16x4*>(tile + off);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = OUT == OUT_BF16 ? bf16_to_f32(x[e]) : f16_to_f32(x[e]);
    }
  };
  // global row of staged row pr in pass `pass`
  auto grow = [&](int pass, int pr) -> int64_t {
    return (int64_t)m0 + (pr / WROWS) * WTM + pass * WROWS + (pr % WROWS);
  };
  // The thread index as a value the compiler cannot see through: the
  // per-chunk offsets below are then computed here, in the epilogue.
  // Otherwise they are loop-invariant for the persistent tile loop, get
  // hoisted to the kernel start and spilled across the K loop, and each
  // reload's vmcnt(0) wait also waits for the memory operation issued just
  // before it, which serialises the epilogue's loads.
  auto opaque_tid = [&]() -> int {
    int t = threadIdx.x;
    asm volatile("" : "+v"(t));
    return t;
  };
  // tile rows of this pass -> global matrix (row stride ld elements)
  // (at most four 16-byte chunks in flight: the GELU epilogue calls this
  // with all accumulators live, and more in flight spill them)
  auto copy_out = [&](int pass, void* dst, int64_t ld, const uint8_t* src = nullptr) {
    const uint8_t* from = src ? src : tile;
    const int tid = opaque_tid();
#pragma unroll 4
    for (int k = 0; k < ROWS_PASS * CPR / NT; ++k) {
      const int idx = tid + k * NT;
      const int pr = idx / CPR, c = idx % CPR;
      const u16x8 x = *reinterpret_cast<const u16x8*>(from + pr * ROWB + ((c ^ (pr & (CPR - 1))) * 16));
      store16((uint8_t*)dst + (grow(pass, pr) * ld + n0) * OB + c * 16, x);
    }
  };
  // copy_out of the whole tile (bf16, 256 x 256, 8 waves) that also writes
  // the tile's column sums of the stored (bf16-rounded) values to row m0/256
  // of p.colsum.  A lane always handles the same 8-column chunk c = tid % 32,
  // rows tid / 32 + 16 k (k = 0..15, summed in that order); lanes l and l + 32
  // of a wave hold the same chunk and are added, then the 8 waves in order
  // through LDS.
  auto copy_out_colsum = [&]() {
    const int tid = opaque_tid();
    float cs[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) cs[e] = 0.0f;
#pragma unroll
    for (int k = 0; k < ROWS_PASS * CPR / NT; ++k) {
      const int idx = tid + k * NT;
      const int pr = idx / CPR, c = idx % CPR;
      const u16x8 x = *reinterpret_cast<const u16x8*>(tile + pr * ROWB + ((c ^ (pr & (CPR - 1))) * 16));
      store16((uint8_t*)p.C + (grow(0, pr) * p.ldc + n0) * OB + c * 16, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) cs[e] += bf16_to_f32(x[e]);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) cs[e] += __shfl_xor(cs[e], 32, 64);
    __syncthreads();  // every lane has read its rows of the tile
    float* red = reinterpret_cast<float*>(tile);  // [8 waves][256 columns]
    const int w = tid >> 6, l = tid & 63;
    if (l < 32) {
#pragma unroll
      for (int e = 0; e < 8; ++e) red[w * BN + l * 8 + e] = cs[e];
    }
    __syncthreads();
    if (tid < BN) {
      float s = red[tid];
#pragma unroll
      for (int ww = 1; ww < NW; ++ww) s += red[ww * BN + tid];
      p.colsum[(int64_t)(m0 / BM) * p.N + n0 + tid] = s;
    }
  };
  // global matrix -> tile rows of this pass, straight into LDS (no VGPRs:
  // the accumulators are live).  Wave instruction q fills the 1 KB at
  // tile + 1024 q, i.e. physical chunks idx = 64 q + lane; the lane fetches
  // the logical chunk stored there.
  auto copy_in = [&](int pass, const void* src, int64_t ld) {
    const int tid = opaque_tid();
    const int wave_id = __builtin_amdgcn_readfirstlane(tid >> 6), ln = tid & 63;
#pragma unroll
    for (int k = 0; k < ROWS_PASS * CPR / NT; ++k) {
      const int q = wave_id + k * NW;
      const int idx = q * 64 + ln;
      const int pr = idx / CPR, c = (idx % CPR) ^ (pr & (CPR - 1));
      __builtin_amdgcn_global_load_lds(
          (glb_void_t*)((const uint8_t*)src + (grow(pass, pr) * ld + n0) * OB + c * 16),
          (lds_void_t*)(tile + q * 1024), 16, 0, 0);
    }
    __builtin_amdgcn_s_waitcnt(0);
  };

  // ACT_ADAMW: the staged rows of this pass are the weight gradient; each
  // 16-byte chunk updates 4 weights (P, M, V read and written, bf16 shadow
  // written), row-contiguous like copy_out.
  auto adam_out = [&](int pass) {
    if constexpr (ACT == ACT_ADAMW) {
      const AdamWScalars sc = adamw_scalars(p.adam.step, p.adam.args);
      const int tid = opaque_tid();
#pragma unroll 4
      for (int k = 0; k < ROWS_PASS * CPR / NT; ++k) {
        const int idx = tid + k * NT;
        const int pr = idx / CPR, c = idx % CPR;
        const f32x4 g = *reinterpret_cast<const f32x4*>(tile + pr * ROWB + ((c ^ (pr & (CPR - 1))) * 16));
        const int64_t e = grow(pass, pr) * p.ldc + n0 + c * 4;
        f32x4 pp = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(p.adam.P + e));
        f32x4 mm = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(p.adam.M + e));
        f32x4 vv = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(p.adam.V + e));
        u16x4 w;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float pj = pp[j], mj = mm[j], vj = vv[j];
          adamw_elem(pj, g[j], mj, vj, sc, p.adam.args);
          pp[j] = pj;
          mm[j] = mj;
          vv[j] = vj;
          w[j] = f32_to_bf16(pj);
        }
        __builtin_nontemporal_store(pp, reinterpret_cast<f32x4*>(p.adam.P + e));
        __builtin_nontemporal_store(mm, reinterpret_cast<f32x4*>(p.adam.M + e));
        __builtin_nontemporal_store(vv, reinterpret_cast<f32x4*>(p.adam.V + e));
        __builtin_nontemporal_store(w, reinterpret_cast<u16x4*>(p.adam.Wb + e));
      }
    }
  };

#pragma unroll
  for (int pass = 0; pass < NPASS; ++pass) {
    if constexpr (ACT == ACT_DGELU) {
      copy_in(pass, p.aux, p.aux_ld);
      __syncthreads();
    }
    if constexpr (ACT == ACT_GELU && !GELU_DUAL) {
      if (p.aux) {  // pre-activation z
#pragma unroll
        for (int jj = 0; jj < JP; ++jj)
#pragma unroll
          for (int i = 0; i < TN; ++i)
#pragma unroll
            for (int g = 0; g < G; ++g) {
              float v[4];
              frag4(pass * JP + jj, i, g, v);
              put4(slot(jj, i, g), v);
            }
        __syncthreads();
        copy_out(pass, p.aux, p.aux_ld);
        __syncthreads();
      }
    }
#pragma unroll
    for (int jj = 0; jj < JP; ++jj)
#pragma unroll
      for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const int off = slot(jj, i, g);
          float v[4];
          frag4(pass * JP + jj, i, g, v);
          if constexpr (ACT == ACT_DGELU) {
            float z[4];
            get4(off, z);  // this lane's own slot: no barrier between read and write
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] *= gelu_tanh_grad_f(z[e]);
          } else if constexpr (ACT == ACT_RELU) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = v[e] > 0.0f ? v[e] : 0.0f;
          } else if constexpr (ACT == ACT_GELU) {
            if constexpr (GELU_DUAL) {
              if (p.aux) put4(REGION + off, v);  // pre-activation z
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = gelu_tanh_f(v[e]);
          }
          put4(off, v);
        }
    __syncthreads();
    if constexpr (GELU_DUAL) {
      if (p.aux) copy_out(pass, p.aux, p.aux_ld, tile + REGION);
      copy_out(pass, p.C, p.ldc);
    } else if constexpr (ACT == ACT_ADAMW) {
      adam_out(pass);
    } else if constexpr (ACT == ACT_DGELU && OUT == OUT_BF16 && NPASS == 1 && CPR == 32 && NT == 512) {
      if (p.colsum)
        copy_out_colsum();
      else
        copy_out(pass, p.C, p.ldc);
    } else {  // (run_gemm sends column-sum launches to the branch above only)
      copy_out(pass, p.C, p.ldc);
    }
    if (pass + 1 < NPASS) __syncthreads();
  }
}

template <int V>
using template_int_t = std::integral_constant<int, V>;

// Schedule of one MFMA sub-step of the NT kernel: MFMA t is followed by its
// FPER fragments' LDS reads (front-loaded, so the last reads still have
// several MFMAs to land before the next sub-step needs them) and by its
// share of the NV loads, spread over the first LSPAN MFMAs (load u after
// MFMA t when t*NV/LSPAN <= u < (t+1)*NV/LSPAN).  sched_group_barrier masks:
// 0x008 MFMA, 0x100 DS read, 0x020 VMEM read.
template <int TM, int TN, int ES, bool AKC, bool BKC, int MS, int LSPAN>
struct NTSched {
  static constexpr int NMF = TM * TN * (ES == 4 ? 4 : 1);  // MFMAs per sub-step
  static_assert(LSPAN >= 1 && LSPAN <= NMF, "loads spread over the sub-step's MFMAs");
  static constexpr int load_lo(int t, int nv) { return t < LSPAN ? t * nv / LSPAN : nv; }
  static constexpr int NFR = TM + TN;                      // fragments per sub-step
  static constexpr int FPER = (NFR + NMF - 1) / NMF;       // fragments per MFMA
  // 16 x 16 blocks (RECYCLE): the MFMAs run A-fragment-major (t -> block
  // (t % TN, t / TN)) and the next sub-step's A fragment j is read into the
  // same registers right after its last MFMA (t = j TN + TN - 1), so only
  // the B fragments are double-buffered; the next B fragment t is read after
  // MFMA t.  Otherwise fragment r (A for r < TM, else B) after MFMA r / FPER.
  static constexpr bool RECYCLE = MS == 16;
  static constexpr int ds_instrs(int lo, int hi) {
    int n = 0;
    constexpr int MN_READS = ES == 4 ? 4 : 2;  // LDS reads of an M/N-contiguous fragment
    for (int r = lo; r < hi && r < NFR; ++r) n += r < TM ? (AKC ? 1 : MN_READS) : (BKC ? 1 : MN_READS);
    return n;
  }
  static constexpr int ds_after(int t) {
    if (!RECYCLE) return ds_instrs(t * FPER, (t + 1) * FPER);
    return (t < TN ? (BKC ? 1 : 2) : 0) + (t % TN == TN - 1 ? (AKC ? 1 : 2) : 0);
  }
  template <bool R, int NV, int T>
  static __device__ __forceinline__ void step() {
    constexpr int nds = R ? ds_after(T) : 0;
    constexpr int vlo = load_lo(T, NV), vhi = load_lo(T + 1, NV);
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    if constexpr (nds > 0) __builtin_amdgcn_sched_group_barrier(0x100, nds, 0);
    if constexpr (vhi > vlo) __builtin_amdgcn_sched_group_barrier(0x020, vhi - vlo, 0);
  }
  template <bool R, int NV, int... T>
  static __device__ __forceinline__ void seq(std::integer_sequence<int, T...>) {
    (step<R, NV, T>(), ...);
  }
  template <bool R, int NV>
  static __device__ __forceinline__ void pin() {
    seq<R, NV>(std::make_integer_sequence<int, NMF>{});
  }
};

// One operand of the NT kernel: BMN rows (the M or N dimension) x BK = 64
// K-elements per stage.
//   KC (K-contiguous, memory [MN][K] with row stride ld): 1 KB LDS blocks of
//     8 MN-rows x 64 K (128 B per row); row r keeps logical 16-byte chunk c
//     at physical chunk c ^ ((r >> 1) & 7), so the 32-row ds_read_b128
//     fragment reads hit all 64 banks.  Slot `lane` of block j is row
//     8j + lane/8, physical chunk lane%8.
//   MN-contiguous (memory [K][MN] with row stride ld): 64 K-rows of BMN
//     elements; row k keeps logical chunk c (8 MN-elements) at physical chunk
//     c ^ nt_mn_swizzle(k).  A fragment (MS MN x 16 or 32 K) is two
//     ds_read_b64_tr_b16 per 16-lane group: lane j points at row k0 + j/4,
//     elements m + 4 (j%4) .. +3, and the transposing read hands lane i the
//     four K values of element m + i.
//   K-contiguous rows are 128 B: the chunk c ^ ((r >> 1) & 7) keeps the 32
//     (or 16) rows of one fragment read on all 64 banks.
// Loads are buffer loads straight into LDS with per-lane offsets fixed for
// the whole K loop (the K advance is the scalar offset); the host checks that
// the bytes a resource spans fit a signed 32-bit offset.
template <bool KC, int BMN, int NW, int ES>
struct NTOperand {
  static constexpr int BYTES = BMN * 128;            // a stage holds 128 B of K per row
  static constexpr int BLOCKS = BYTES / 1024 / NW;   // 1 KB load blocks per wave
  static constexpr int ROWB = BMN * ES;              // MN-contiguous row bytes
  static constexpr int CPR = ROWB / 16;              // chunks per MN-contiguous row
  static_assert(BYTES % (1024 * NW) == 0, "load blocks must split evenly over waves");
  static_assert(KC || CPR >= 16 || (ES == 2 && CPR == 8), "MN-contiguous tiles: >= 16 chunks per row, or 8 (16-bit)");

  i32x4_t rsrc;
  int voff[BLOCKS];
  int soff_step;  // scalar byte offset per K-step
};

// EDGE: the operand has mn_total rows (M/N-contiguous: columns) and K K-rows;
// what lies behind them is not read and counts as zero.
template <bool KC, int BMN, int NW, int ES, int MS, bool EDGE = false>
__device__ __forceinline__ void nt_operand_init(NTOperand<KC, BMN, NW, ES>& o, const void* X, int64_t ld,
                                                int mn0, int K, int lane, int wave, int mn_total = 0) {
  const uint8_t* Xb = static_cast<const uint8_t*>(X);
  if constexpr (KC) {
    const int rows = !EDGE || mn_total - mn0 > BMN ? BMN : mn_total - mn0;
    o.rsrc = buffer_rsrc(Xb + (int64_t)mn0 * ld * ES, (uint32_t)((int64_t)rows * ld * ES));
    const int r_in = lane >> 3;
    const int cl_even = (lane & 7) ^ (r_in >> 1);
    const int cl_odd = (lane & 7) ^ ((4 + (r_in >> 1)) & 7);
#pragma unroll
    for (int t = 0; t < o.BLOCKS; ++t) {
      const int j = wave + t * NW;
      o.voff[t] = (j * 8 + r_in) * (int)ld * ES + ((j & 1) ? cl_odd : cl_even) * 16;
    }
    o.soff_step = 128;
  } else {
    constexpr int CPR = NTOperand<KC, BMN, NW, ES>::CPR;
    constexpr int RPB = 64 / CPR;  // rows per 1 KB block
    int64_t span = (int64_t)K * ld;
    if constexpr (EDGE) span = K > 0 ? span - ld + (mn_total - mn0) : 0;
    o.rsrc = buffer_rsrc(Xb + (int64_t)mn0 * ES, (uint32_t)(span * ES));
#pragma unroll
    for (int t = 0; t < o.BLOCKS; ++t) {
      const int q = wave + t * NW;
      const int k = q * RPB + lane / CPR;
      const int c = (lane % CPR) ^ nt_mn_swizzle<MS, ES, CPR>(k);
      o.voff[t] = k * (int)ld * ES + c * 16;
    }
    o.soff_step = 128 * (int)ld;  // 128 / ES K-rows per stage
  }
}

// The epilogues of ACT_LX_* (linear_xent.hip).
template <int OUT, int ACT, int BM, int BN, int WM, int WN, int STAGE_BYTES, int MS>
__device__ void lx_epilogue(const NTParams& p, nt_acc_t<MS> (&acc)[BN / WN / MS][BM / WM / MS], uint8_t* smem,
                            int m0, int n0);

// Persistent tiles (one workgroup per CU looping over tiles) for the 8-wave
// 256 x 256 configuration; the 4-wave one keeps one tile per workgroup: its
// 256 accumulators per lane leave no room for the registers that a tile loop
// carries through the epilogue (they spill to scratch and cost more than the
// overlap gains).
constexpr bool nt_persistent(int BM, int BN, int WM, int WN) {
  return BM == 256 && BN == 256 && WM * WN == 8;
}

// S: LDS stages.  Two for the large tiles (their K-step's MFMA work covers a
// load's latency); small tiles, whose K-step is a few hundred cycles of MFMA
// work, keep S - 1 K-steps of loads in flight.
template <int IN, int OUT, int ACT, int BM, int BN, int WM, int WN, bool AKC, bool BKC, int S = 2>
__global__ __launch_bounds__(64 * WM * WN) void gemm_nt_kernel(NTParams p) {
  static_assert(S == 2 || S == 4 || S == 8, "stages: 2, 4 or 8");
  constexpr int ES = IN == IN_F32 ? 4 : 2;  // element bytes
  // MFMA block: 16 x 16 x 32 for 16-bit operands, 32 x 32 x 2 for fp32
  constexpr int MS = ES == 2 ? 16 : 32;
  constexpr int KS = MS == 16 ? 2 : 4;  // MFMA sub-steps per K-step
  constexpr int CPS = 64 / MS;          // 16-byte chunks of a 128-byte K-row per sub-step
  constexpr int KPS = ES == 4 ? 8 : 16 * CPS / 2;  // K-rows of an MN-contiguous stage per sub-step
  constexpr int NW = WM * WN;
  constexpr int WTM = BM / WM, WTN = BN / WN;
  constexpr int TM = WTM / MS, TN = WTN / MS;
  constexpr int A_BYTES = BM * 128, B_BYTES = BN * 128;  // 128 B of K per row and stage
  constexpr int STAGE = A_BYTES + B_BYTES;
  constexpr bool LX = ACT >= ACT_LX_STATS;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[S * STAGE];
  if constexpr (LX) {
    const int rows = p.lx.n[0];
    if (p.lx.rows_are_k) {
      p.K = rows;
    } else {
      p.M = rows;
      p.tiles_m = (rows + BM - 1) / BM;
    }
  }
  int shares = 1, k_share = 0;
  if constexpr (ACT == ACT_LX_SLAB) {
    shares = p.lx.shares[0];
    k_share = lx_share_k(p.lx.k_piece, shares);
  }

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = wave / WN, wn = wave % WN;
  const int wave_s = __builtin_amdgcn_readfirstlane(wave);
  int m0 = 0, n0 = 0;
  NTOperand<AKC, BM, NW, ES> opa;
  NTOperand<BKC, BN, NW, ES> opb;

  // Load u of the wave for K-step kt into stage `stage`: 1 KB direct-to-LDS
  // block u (A blocks first).  With an M/N-contiguous operand the loads are
  // issued as inline asm (no compiler waits in front of the transposing
  // reads); K-contiguous kernels use the intrinsic, which the scheduler
  // places by itself.
  constexpr bool ASM_LDS = !(AKC && BKC);
  constexpr int NVM = opa.BLOCKS + opb.BLOCKS;  // loads per wave and K-step
  // ACT_LX_*, K-contiguous: the K-step that K does not fill is taken first, as
  // K-step nk of 1 .. nk, with B's chunks behind K sent out of bounds (16 bytes
  // divide a row; A has zeros there).
  int k_shift = 0, k_out = 0;
  if constexpr (LX && AKC && BKC) {
    static_assert(NW % 2 == 0, "a wave's blocks have one parity");
    const int rest = p.K * ES % 128, c = (lane & 7) ^ ((4 * (wave & 1) + (lane >> 4)) & 7);
    k_shift = rest > 0 ? 1 : 0;
    k_out = rest > 0 && c * 16 >= rest ? (int)0x80000000 : 0;
  }
  auto load_one = [&](int kt, int stage, int u, auto PAD, int out = 0) {
    uint8_t* base = smem + stage * STAGE;
    const bool is_a = u < opa.BLOCKS;
    uint8_t* dst = is_a ? base + (wave_s + u * NW) * 1024 : base + A_BYTES + (wave_s + (u - opa.BLOCKS) * NW) * 1024;
    const i32x4_t rsrc = is_a ? opa.rsrc : opb.rsrc;
    const int voff = is_a ? opa.voff[u] : opb.voff[u - opa.BLOCKS];
    const int soff = (kt - k_shift) * (is_a ? opa.soff_step : opb.soff_step);
    if constexpr (ASM_LDS)
      asm_buffer_load_lds<decltype(PAD)::value>(rsrc, (uint32_t)(uintptr_t)dst, voff, soff);
    else
      raw_buffer_load_lds(rsrc, (__attribute__((address_space(3))) unsigned*)dst, 16, voff | out, soff, 0, 0);
  };
  auto issue_loads = [&](int kt, int stage) {
#pragma unroll
    for (int u = 0; u < NVM; ++u) load_one(kt, stage, u, std::true_type{});
  };

  nt_acc_t<MS> acc[TN][TM];

  // Fragment addresses.  K-contiguous: row offset of the lane's MN-row plus
  // the swizzled chunk of (sub-step, lane group).  MN-contiguous: the lane's
  // K-row within a sub-step and its swizzled column bytes (loop invariant).
  // A lane of an MS x MS block holds MN-row fr and K chunk fh of the
  // sub-step (8 K per 16-byte chunk).
  const int fr = lane % MS, fh = lane / MS;
  const int rsw = (fr >> 1) & 7;  // fragment rows start at multiples of MS
  const int g16 = (lane >> 4) & 3, i16 = lane & 15;
  // 32 x 32: groups 0/1 take MN + 0/16 of K-rows 0-7, groups 2/3 K-rows
  // 8-15; 16 x 16: group g takes K-rows 8 g .. 8 g + 7 of the same 16 MN
  const int tr_row = MS == 32 ? (8 * (g16 >> 1) + (i16 >> 2)) : (8 * g16 + (i16 >> 2));
  // byte offset of the lane's 8-byte piece in a K-row of `cpr` chunks
  auto tr_col = [&](int mb, auto CPR_) {
    constexpr int cpr = decltype(CPR_)::value;
    if constexpr (MS == 32)
      return ((((mb >> 3) ^ (4 * ((i16 >> 2) & 3))) + 2 * (g16 & 1) + ((i16 >> 1) & 1)) * 16) + 8 * (i16 & 1);
    else
      return ((((mb >> 3) ^ nt_mn_swizzle<MS, 2, cpr>(tr_row)) + ((i16 >> 1) & 1)) * 16) + 8 * (i16 & 1);
  };
  // fp32 M/N-contiguous: lane (fr, fh) holds element mb + fr of K-rows
  // 4 fh .. 4 fh + 3 of the sub-step (four 4-byte reads, one per K-row);
  // the row swizzle of those rows is 8 fh
  auto mn32_off = [&](int mb, int rowb) {
    const int m = mb + fr;
    return 4 * fh * rowb + (((m >> 2) ^ (8 * fh)) * 16) + (m & 3) * 4;
  };
  int a_off[TM], b_off[TN];
#pragma unroll
  for (int j = 0; j < TM; ++j) {
    const int mb = wm * WTM + j * MS;
    if constexpr (AKC) a_off[j] = (mb + fr) * 128;
    else a_off[j] = ES == 4 ? mn32_off(mb, BM * ES) : tr_row * (BM * 2) + tr_col(mb, template_int_t<BM * 2 / 16>{});
  }
#pragma unroll
  for (int i = 0; i < TN; ++i) {
    const int nb = wn * WTN + i * MS;
    if constexpr (BKC) b_off[i] = A_BYTES + (nb + fr) * 128;
    else b_off[i] = A_BYTES + (ES == 4 ? mn32_off(nb, BN * ES) : tr_row * (BN * 2) + tr_col(nb, template_int_t<BN * 2 / 16>{}));
  }

  typedef short v4i16 __attribute__((ext_vector_type(4)));
  auto tr_frag = [&](const uint8_t* addr, int rowb) -> u16x8 {
    if constexpr (ES == 4) {  // fp32: four K-rows, one float each
      f32x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = *reinterpret_cast<const float*>(addr + e * rowb);
      return __builtin_bit_cast(u16x8, v);
    } else {
      const v4i16 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4i16*)addr);
      const v4i16 hi =
          __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4i16*)(addr + 4 * rowb));
      u16x8 f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f[e] = (uint16_t)lo[e];
        f[e + 4] = (uint16_t)hi[e];
      }
      return f;
    }
  };

  u16x8 fa[2][TM], fb[2][TN];
  auto read_frags = [&](const uint8_t* st, int kk, int buf) {
    const int chunk = ((kk * CPS + fh) ^ rsw) * 16;
#pragma unroll
    for (int j = 0; j < TM; ++j) {
      const int ab = MS == 16 ? 0 : buf;
      if constexpr (AKC) fa[ab][j] = *reinterpret_cast<const u16x8*>(st + a_off[j] + chunk);
      else fa[ab][j] = tr_frag(st + a_off[j] + kk * KPS * (BM * ES), BM * ES);
    }
#pragma unroll
    for (int i = 0; i < TN; ++i) {
      if constexpr (BKC) fb[buf][i] = *reinterpret_cast<const u16x8*>(st + b_off[i] + chunk);
      else fb[buf][i] = tr_frag(st + b_off[i] + kk * KPS * (BN * ES), BN * ES);
    }
  };
  // Single operations of the pipeline, emitted one by one in the order the
  // schedule below pins (the compiler keeps LDS-writing loads and LDS reads
  // in program order, so the order has to be written out).
  //   fragment f: f < TM is A fragment f, else B fragment f - TM (one
  //     ds_read_b128, or two ds_read_b64_tr_b16 for an M/N-contiguous tile);
  //     with RECYCLE (NTSched) the A fragments use register set 0 only;
  //   MFMA t: block (i, j) = (t / TM % TN, t % TM), or (t % TN, t / TN) with
  //     RECYCLE; fp32 runs 4 MFMAs per block and sub-step, t / (TM * TN)
  //     selecting the fragment element;
  //   load u: 1 KB direct-to-LDS block u of the wave (A blocks first).
  // The 8-wave tiles with 16-bit operands spread a K-step's loads over the
  // first 3/4 of the first sub-step's MFMAs, the others over all of them
  // (step 2.85 -> 2.79 ms, same bits; spans of 5/8 and 7/8, a later start,
  // or loads in both sub-steps were slower, and 3/4 on the 4-wave tiles
  // slowed 8192^3).
  constexpr int NMF_ = TM * TN * (ES == 4 ? 4 : 1);
  using Sched = NTSched<TM, TN, ES, AKC, BKC, MS, NW == 8 && ES == 2 ? NMF_ * 3 / 4 : NMF_>;
  constexpr bool RECYCLE = Sched::RECYCLE;
  auto read_one = [&](const uint8_t* st, int kk, int buf, int f) {
    const int chunk = ((kk * CPS + fh) ^ rsw) * 16;
    if (f < TM) {
      const int ab = RECYCLE ? 0 : buf;
      if constexpr (AKC) fa[ab][f] = *reinterpret_cast<const u16x8*>(st + a_off[f] + chunk);
      else fa[ab][f] = tr_frag(st + a_off[f] + kk * KPS * (BM * ES), BM * ES);
    } else {
      const int i = f - TM;
      if constexpr (BKC) fb[buf][i] = *reinterpret_cast<const u16x8*>(st + b_off[i] + chunk);
      else fb[buf][i] = tr_frag(st + b_off[i] + kk * KPS * (BN * ES), BN * ES);
    }
  };
  auto mfma_one = [&](int buf, int t) {
    const int i = RECYCLE ? t % TN : (t / TM) % TN, j = RECYCLE ? t / TN : t % TM;
    if constexpr (MS == 16) {
      acc[i][j] = mfma16<IN>(reinterpret_cast<const uint16_t*>(&fb[buf][i]),
                             reinterpret_cast<const uint16_t*>(&fa[0][j]), acc[i][j]);
    } else if constexpr (ES == 2) {
      acc[i][j] = mfma32<IN>(reinterpret_cast<const uint16_t*>(&fb[buf][i]),
                             reinterpret_cast<const uint16_t*>(&fa[buf][j]), acc[i][j]);
    } else {
      const int e = t / (TM * TN);
      const float a = reinterpret_cast<const float*>(&fb[buf][i])[e];
      const float b = reinterpret_cast<const float*>(&fa[buf][j])[e];
      acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, acc[i][j], 0, 0, 0);
    }
  };
  constexpr int NMF = Sched::NMF, NFR = Sched::NFR, FPER = Sched::FPER;
  // One sub-step: the MFMAs on fragment buffer `buf`; when R, the fragments
  // of sub-step rkk of stage `rst` into buffer rbuf (front-loaded, FPER per
  // MFMA); loads [VLO, VHI) of K-step lkt into stage lst, spread evenly.
  auto substep = [&](auto R, auto VLO, auto VHI, int buf, const uint8_t* rst, int rkk, int rbuf, int lkt,
                     int lst) {
    constexpr int vlo = decltype(VLO)::value, vhi = decltype(VHI)::value, nv = vhi - vlo;
#pragma unroll
    for (int t = 0; t < NMF; ++t) {
      mfma_one(buf, t);
      if constexpr (decltype(R)::value) {
        if constexpr (RECYCLE) {
          if (t < TN) read_one(rst, rkk, rbuf, TM + t);
          if (t % TN == TN - 1) read_one(rst, rkk, rbuf, t / TN);
        } else {
#pragma unroll
          for (int q = 0; q < FPER; ++q)
            if (t * FPER + q < NFR) read_one(rst, rkk, rbuf, t * FPER + q);
        }
      }
      if constexpr (nv > 0) {
#pragma unroll
        for (int u = vlo + Sched::load_lo(t, nv); u < vlo + Sched::load_lo(t + 1, nv); ++u)
          load_one(lkt, lst, u, std::false_type{});
      }
    }
    Sched::template pin<decltype(R)::value, ASM_LDS ? 0 : nv>();  // asm loads are in no sched group
  };
  using Rd = std::true_type;
  using NoRd = std::false_type;
  template_int_t<0> z;

  // Pipeline.  A K-step (128 bytes of K per row) has KS sub-steps (four of
  // 32 x 32 x 16 or 32 x 32 x 2 MFMAs, or two of 16 x 16 x 32); the
  // fragments of sub-step s+1 are read during the MFMAs of sub-step s, from
  // two register sets.  The body of the K loop starts with the K-step's only
  // barrier: after it the stage of K-step kt+1 is visible to every wave and
  // the stage of K-step kt is read by none, so the loads of K-step kt+2
  // refill it.  The body then runs the last sub-step of kt (its fragments are
  // already in registers) and the other sub-steps of kt+1, with the loads of
  // kt+2 spread over the first half of the body: issued all at once after the
  // barrier they back up the address queue and stall the MFMA issue, and
  // issued later they have too little time left before the next wait.
  // Tiles: the grid covers all tiles (one per workgroup), or, persistent,
  // one workgroup per CU loops over tiles blockIdx.x + q * gridDim.x, so that
  // the global stores of a tile's epilogue drain while the next tile's loads
  // and MFMAs run.  With a grid that is a multiple of 8, tile % 8 is the
  // workgroup's XCD, as the remap in tile_coords_of assumes.
  int total_tiles = p.tiles_m * p.tiles_n;
  constexpr bool PERSIST = nt_persistent(BM, BN, WM, WN) || ACT == ACT_LX_SLAB;
  const int tiles_of_share = total_tiles;
  NTParams q = p;  // ACT_LX_SLAB: of the tile's share
  if constexpr (ACT == ACT_LX_SLAB) total_tiles *= shares;
  for (int tile = blockIdx.x; tile < total_tiles; tile += gridDim.x) {
  {
    int tm_i, tn_i, in_share = tile;
    if constexpr (ACT == ACT_LX_SLAB) {  // (A K-contiguous, B N-contiguous)
      const int share = tile / tiles_of_share, k0 = share * k_share;
      if (k0 >= p.K) continue;  // a short piece has fewer shares
      in_share = tile - share * tiles_of_share;
      q.K = p.K - k0 < k_share ? p.K - k0 : k_share;
      q.A = (const uint8_t*)p.A + (int64_t)k0 * ES;
      q.B = (const uint8_t*)p.B + (int64_t)k0 * p.ldb * ES;
      q.C = (float*)p.C + (int64_t)share * (p.tiles_m * BM) * p.ldc;  // (slabs of whole tiles)
      q.lx.add = k0 < p.lx.k_before;
    }
    tile_coords_of<LX>(in_share, p.tiles_m, p.tiles_n, tm_i, tn_i);
    m0 = tm_i * BM;
    n0 = tn_i * BN;
    if constexpr (ACT != ACT_ADAMW && !LX) {
      // A last tile that would pass M or N is moved back to end there: it
      // computes rows or columns of its neighbour again, with the same bits
      // (an output's K order does not depend on its place in a tile).
      m0 = m0 < p.M - BM ? m0 : p.M - BM;
      n0 = n0 < p.N - BN ? n0 : p.N - BN;
    }
  }
  nt_operand_init<AKC, BM, NW, ES, MS, LX>(opa, q.A, p.lda, m0, q.K, lane, wave, p.lx.a_mn);
  nt_operand_init<BKC, BN, NW, ES, MS, LX>(opb, q.B, p.ldb, n0, q.K, lane, wave, p.lx.b_mn);
#pragma unroll
  for (int i = 0; i < TN; ++i)
#pragma unroll
    for (int j = 0; j < TM; ++j)
#pragma unroll
      for (int r = 0; r < (MS == 16 ? 4 : 16); ++r) acc[i][j][r] = 0.0f;

  int nk = q.K / (128 / ES);
  if constexpr (LX) nk = q.K > 0 ? (q.K + 128 / ES - 1) / (128 / ES) : 1;
  constexpr int L1 = NVM / 2;  // with four sub-steps: loads in the first of the two
  // Wait until at most n K-steps of this wave's loads are in flight (and its
  // fragment reads are done); n < S - 1.
  auto wait_steps = [&](int n) {
    if constexpr (S > 2) {
      if (n >= 6) { wait_vm_lgkm0<6 * NVM>(); return; }
      if (n == 5) { wait_vm_lgkm0<5 * NVM>(); return; }
      if (n == 4) { wait_vm_lgkm0<4 * NVM>(); return; }
      if (n == 3) { wait_vm_lgkm0<3 * NVM>(); return; }
      if (n == 2) { wait_vm_lgkm0<2 * NVM>(); return; }
      if (n == 1) { wait_vm_lgkm0<NVM>(); return; }
    }
    __builtin_amdgcn_s_waitcnt(0);
  };
  if constexpr (LX && AKC && BKC) {
#pragma unroll
    for (int u = 0; u < NVM; ++u) load_one(k_shift * nk, 0, u, std::false_type{}, u < opa.BLOCKS ? 0 : k_out);
  } else {
    issue_loads(0, 0);
  }
  if constexpr (S > 2) {
    // K-steps 1 .. S - 2 go out before the first wait
    for (int q = 1; q < S - 1 && q < nk; ++q) issue_loads(q, q);
    wait_steps((nk - 1 < S - 2 ? nk - 1 : S - 2));
    barrier_keep_loads();
  } else {
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
  }
  if (S - 1 < nk) issue_loads(S - 1, S - 1);
  read_frags(smem, 0, 0);
  if constexpr (KS == 4) {
    substep(Rd{}, z, z, 0, smem, 1, 1, 0, 0);
    substep(Rd{}, z, z, 1, smem, 2, 0, 0, 0);
    substep(Rd{}, z, z, 0, smem, 3, 1, 0, 0);
  } else {
    substep(Rd{}, z, z, 0, smem, 1, 1, 0, 0);
  }
  int kt = 0;
  for (; kt + S < nk; ++kt) {
    // own loads of K-step kt+1 and fragment reads done; K-steps kt+2 ..
    // kt+S-1 may still be in flight
    if constexpr (S > 2) {
      wait_vm_lgkm0<(S - 2) * NVM>();
      barrier_keep_loads();
    } else {
      __builtin_amdgcn_s_waitcnt(0);
      __syncthreads();
    }
    const uint8_t* nx = smem + ((kt + 1) % S) * STAGE;
    const int ls = kt % S;  // the stage of K-step kt, free after the barrier, takes K-step kt+S
    if constexpr (KS == 4) {
      substep(Rd{}, z, template_int_t<L1>{}, 1, nx, 0, 0, kt + S, ls);
      substep(Rd{}, template_int_t<L1>{}, template_int_t<NVM>{}, 0, nx, 1, 1, kt + S, ls);
      substep(Rd{}, z, z, 1, nx, 2, 0, 0, 0);
      substep(Rd{}, z, z, 0, nx, 3, 1, 0, 0);
    } else {
      // two sub-steps of twice the MFMAs: the loads of K-step kt+S over the first
      substep(Rd{}, z, template_int_t<NVM>{}, 1, nx, 0, 0, kt + S, ls);
      substep(Rd{}, z, z, 0, nx, 1, 1, 0, 0);
    }
  }
  if constexpr (S > 2) {
    for (; kt + 2 < nk; ++kt) {  // nothing left to load: K-steps kt+2 .. nk-1 in flight
      wait_steps(nk - 2 - kt);
      barrier_keep_loads();
      const uint8_t* nx = smem + ((kt + 1) % S) * STAGE;
      if constexpr (KS == 4) {
        substep(Rd{}, z, z, 1, nx, 0, 0, 0, 0);
        substep(Rd{}, z, z, 0, nx, 1, 1, 0, 0);
        substep(Rd{}, z, z, 1, nx, 2, 0, 0, 0);
        substep(Rd{}, z, z, 0, nx, 3, 1, 0, 0);
      } else {
        substep(Rd{}, z, z, 1, nx, 0, 0, 0, 0);
        substep(Rd{}, z, z, 0, nx, 1, 1, 0, 0);
      }
    }
  }
  if constexpr (ASM_LDS) {
    // The asm loads are hidden from the compiler's hazard tracking: once the
    // loop has issued its last one, their lane offsets are dead to it and
    // their registers could be reused while those loads are in flight.  Wait
    // for them here and keep the offsets live up to this point.
    __builtin_amdgcn_s_waitcnt(0);
#pragma unroll
    for (int t = 0; t < opa.BLOCKS; ++t) asm volatile("" ::"v"(opa.voff[t]));
#pragma unroll
    for (int t = 0; t < opb.BLOCKS; ++t) asm volatile("" ::"v"(opb.voff[t]));
  }
  if (kt + 1 < nk) {
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    const uint8_t* nx = smem + ((kt + 1) % S) * STAGE;
    if constexpr (KS == 4) {
      substep(Rd{}, z, z, 1, nx, 0, 0, 0, 0);
      substep(Rd{}, z, z, 0, nx, 1, 1, 0, 0);
      substep(Rd{}, z, z, 1, nx, 2, 0, 0, 0);
      substep(Rd{}, z, z, 0, nx, 3, 1, 0, 0);
    } else {
      substep(Rd{}, z, z, 1, nx, 0, 0, 0, 0);
      substep(Rd{}, z, z, 0, nx, 1, 1, 0, 0);
    }
  }
  substep(NoRd{}, z, z, 1, nullptr, 0, 0, 0, 0);

  __syncthreads();  // every wave is done reading the last stage
  if constexpr (ACT == ACT_LX_SLAB) {
    if (shares == 1 && q.lx.direct) {
      q.C = q.lx.direct;
      q.ldc = q.lx.ld_direct;
      lx_epilogue<OUT, ACT_LX_OUT, BM, BN, WM, WN, 2 * STAGE, MS>(q, acc, smem, m0, n0);
    } else {
      q.ldc = p.ldc;
      lx_epilogue<OUT_F32, ACT, BM, BN, WM, WN, 2 * STAGE, MS>(q, acc, smem, m0, n0);
    }
  } else if constexpr (LX)
    lx_epilogue<OUT, ACT, BM, BN, WM, WN, 2 * STAGE, MS>(q, acc, smem, m0, n0);
  else
    nt_epilogue_staged<OUT, ACT, BM, BN, WM, WN, 2 * STAGE, MS>(p, acc, smem, m0, n0);
  if constexpr (!PERSIST) break;  // one tile per workgroup: no loop-carried registers
  __syncthreads();  // the staged tile is read out before the next tile's loads refill the stages
  }
}

// Compute units of the current device (cached per device; 0 if unknown).
int device_cu_count() {
  static int cached[64] = {0};
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 0;
  if (cached[dev] == 0) {
    int n = 0;
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess) return 0;
    cached[dev] = n;
  }
  return cached[dev];
}

}  // namespace

}  // namespace aicf::hip
