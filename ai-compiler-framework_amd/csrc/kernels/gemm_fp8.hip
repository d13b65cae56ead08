// Matrix product in 8-bit floating point with a f32 scale for each block of
// 128 along K, on the MFMA matrix cores.
//
//   C[m,n] = sum_b SA[m,b] SB[n,b] ( sum over k in block b of A[m,k] B[n,k] ) + bias[n]
//
// A [M, K] and B [N, K] are e4m3 or e5m2 each, K-contiguous; their scales are
// by rows ([M, ceil(K/128)]) or by blocks ([ceil(M/128), ceil(K/128)]).  SA SB is
// taken first: one multiplication for a block's 4 results a lane, where scaling
// each result twice would cost 3 more (39 and 49 cycles an MFMA, below).
//
// A K-step is one scale block, 128 bytes a row: its products start from zero,
// and the four results a lane are added to the f32 accumulators with one
// multiply-add each by SA SB.
//
// 16-bit outputs: one v_mfma_f32_16x16x128_f8f6f4 a block.  That instruction
// (and every other 8-bit one) adds the products of 8 consecutive K after
// aligning them to the largest, and keeps 13 bits below its exponent; the groups
// of 8 are added in f32.  So a result is off by up to 7 2^-13 of the sum of the
// groups' largest products, whatever cancels behind them.  512 x 512 x 4096,
// quantised values, error in the 2-norm relative to the result's, f16 and bf16
// outputs (their rounding alone: 2.07e-4, 1.66e-3):
//   normally distributed               2.08e-4  1.66e-3  (unrounded 1.5e-5)
//   1% of A's channels 1000 x larger   2.19e-4  1.66e-3
//   A log-normal, sigma 2              2.15e-4  1.65e-3
//   pairs that cancel to some 2%       3.16e-4  1.68e-3
// The last, and single results near 0, show it.  f32 outputs have f32 sums.
// f32 outputs: the codes become bf16, which holds both 8-bit types exactly, and
// four v_mfma_f32_16x16x32_bf16 make the block's products and f32 sums (off by
// 1e-8), at half the rate.
//
// The B rows are the MFMA's first operand, so a lane holds 4 consecutive
// columns of one output row.  Which 32 of the 128 K a lane's 8 registers hold
// does not matter as long as it is the same for both operands: the two 16-byte
// chunks g and g + 4 of a row for the lane group g = lane / 16.
//
// No counterpart in the reference.
#include "../common/gemm_types.hpp"
#include "../common/head_util.hpp"
#include "../common/lds_load.hpp"

#include <type_traits>

namespace aicf::hip {

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef uint64_t u64x2_t __attribute__((ext_vector_type(2)));
typedef uint64_t u64x2_a1 __attribute__((ext_vector_type(2), aligned(1)));

struct Fp8Gemm {
  const uint8_t* A;
  const uint8_t* B;
  const float* SA;
  const float* SB;
  const float* bias;
  void* C;
  int64_t lda, ldb, ldc;
  int64_t sa_r, sa_c, sb_r, sb_c;  // scale strides
  int M, N, K;
  int sa_sh, sb_sh;  // row -> scale row: 0 by rows, 7 by blocks
  int out;           // ElemKind
  int tiles_m, tiles_n;
};

// A lane's 32 codes of a row: as they are, or as bf16.  F: 0 e4m3, 1 e5m2.
template <int F, bool EXACT>
struct Frag {
  i32x8 w;
  __device__ __forceinline__ void set(u32x4_t lo, u32x4_t hi) {
    w = i32x8{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
  }
};
template <int F>
struct Frag<F, true> {
  u32x4_t w[4];
  __device__ __forceinline__ void set(u32x4_t lo, u32x4_t hi) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t x = e < 4 ? lo[e] : hi[e - 4];
      bf16x2_t p, q;
      if constexpr (F == 0) {
        p = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.0f, false);
        q = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.0f, true);
      } else {
        p = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(x, 1.0f, false);
        q = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(x, 1.0f, true);
      }
      w[e >> 1][(e & 1) * 2] = __builtin_bit_cast(uint32_t, p);
      w[e >> 1][(e & 1) * 2 + 1] = __builtin_bit_cast(uint32_t, q);
    }
  }
};

// The products of 16 rows of B and 16 of A over one block of K.
template <int AF, int BF>
__device__ __forceinline__ f32x4 mfma_block(const Frag<BF, false>& b, const Frag<AF, false>& a) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b.w, a.w, f32x4{0.0f, 0.0f, 0.0f, 0.0f}, BF, AF, 0, 0, 0,
                                                          0);
}
template <int AF, int BF>
__device__ __forceinline__ f32x4 mfma_block(const Frag<BF, true>& b, const Frag<AF, true>& a) {
  typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
  f32x4 d = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int q = 0; q < 4; ++q)
    d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, b.w[q]),
                                                __builtin_bit_cast(bf16x8_t, a.w[q]), d, 0, 0, 0);
  return d;
}

// 4 outputs of a 16-bit type.
__device__ __forceinline__ uint2 pack_out4(int out, const f32x4& v) {
  if (out == EL_BF16) return uint2{f32x2_to_bf16x2(v[0], v[1]), f32x2_to_bf16x2(v[2], v[3])};
  return uint2{f32_to_f16(v[0]) | (uint32_t)f32_to_f16(v[1]) << 16,
               f32_to_f16(v[2]) | (uint32_t)f32_to_f16(v[3]) << 16};
}

// 4 consecutive outputs of a row, n of them inside.
__device__ __forceinline__ void store_out4(void* C, int out, int64_t at, const f32x4& v, int n) {
  typedef uint32_t u32x2_a2 __attribute__((ext_vector_type(2), aligned(2)));
  if (out == EL_F32) {
    float* p = static_cast<float*>(C) + at;
    if (n >= 4) {
      *reinterpret_cast<f32x4_a4*>(p) = v;
    } else {
#pragma unroll
      for (int e = 0; e < 3; ++e)
        if (e < n) p[e] = v[e];
    }
    return;
  }
  uint16_t* p = static_cast<uint16_t*>(C) + at;
  const uint2 w = pack_out4(out, v);
  if (n >= 4) {
    *reinterpret_cast<u32x2_a2*>(p) = u32x2_a2{w.x, w.y};
  } else {
    if (n > 0) p[0] = (uint16_t)w.x;
    if (n > 1) p[1] = (uint16_t)(w.x >> 16);
    if (n > 2) p[2] = (uint16_t)w.y;
  }
}

// 16 bytes of a row from K position k on, zero from K on, at any alignment.  A
// chunk that would pass K is moved back to end there and shifted into place.
__device__ __forceinline__ u32x4_t load_chunk(const uint8_t* row, int k, int K) {
  u64x2_t w = {0, 0};
  if (k < K) {
    if (K >= 16) {
      const int at = min(k, K - 16), s = (k - at) * 8;
      w = *reinterpret_cast<const u64x2_a1*>(row + at);
      if (s >= 64) w = u64x2_t{w[1] >> (s - 64), 0};
      else if (s > 0) w = u64x2_t{(w[0] >> s) | (w[1] << (64 - s)), w[1] >> s};
    } else {
#pragma unroll 1
      for (int e = K - 1; e >= k; --e) w = u64x2_t{(w[0] << 8) | row[e], (w[1] << 8) | (w[0] >> 56)};
    }
  }
  return __builtin_bit_cast(u32x4_t, w);
}

// Byte of chunk c of a row in a stage of 128-byte rows: 16 rows' equal chunks
// fall on 16 different 16-byte slots of the 256 bytes of all banks.
__device__ __forceinline__ int stage_byte(int row, int c) { return row * 128 + ((c ^ ((row >> 1) & 7)) << 4); }

template <int F, bool EXACT>
__device__ __forceinline__ Frag<F, EXACT> read_frag(const uint8_t* st, int row, int g) {
  Frag<F, EXACT> f;
  f.set(*reinterpret_cast<const u32x4_t*>(st + stage_byte(row, g)),
        *reinterpret_cast<const u32x4_t*>(st + stage_byte(row, g + 4)));
  return f;
}

// ---------------------------------------------------------------------------
// Any sizes, strides and alignments: tiles go through registers into one of
// two LDS stages; the loads of the next block are in flight during this one's
// products.  Rows past M or N read the last row again (not stored), K past the
// end is zero in both operands.
// 4096 x 4096 x 4095, rows at any byte: bf16 193 us, f32 258 (64 x 64 tiles 316
// and 334, 128 x 64 278 and 274); 1001 x 1003 x 785 f16 9.4 on 64 x 64 (19.4 on 128
// x 128).  Bound by the loads: a 16-byte load that crosses a line counts twice.
// With all registers of a SIMD to one wave nothing spills, and it takes 263.
// ---------------------------------------------------------------------------
template <int BM, int BN, int WM, int WN, int AF, int BF, bool BROW, bool EXACT>
__global__ __launch_bounds__(64 * WM * WN, 2) void gemm_fp8_kernel(Fp8Gemm p) {
  constexpr int T = 64 * WM * WN;
  constexpr int TM = BM / WM / 16, TN = BN / WN / 16;
  constexpr int CA = BM * 8 / T, CB = BN * 8 / T;  // 16-byte chunks a thread
  static_assert(CA * T == BM * 8 && CB * T == BN * 8, "chunks split evenly");
  __shared__ __attribute__((aligned(16))) uint8_t smem[2][(BM + BN) * 128];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int wm = wave / WN, wn = wave % WN, r = lane & 15, g = lane >> 4;
  const int tile_m = blockIdx.x % p.tiles_m, tile_n = blockIdx.x / p.tiles_m;
  const int m0 = tile_m * BM, n0 = tile_n * BN;
  const int nkb = (p.K + 127) / 128;

  const uint8_t* pa[CA];
  const uint8_t* pb[CB];
#pragma unroll
  for (int i = 0; i < CA; ++i) pa[i] = p.A + (int64_t)min(m0 + (t >> 3) + i * (T / 8), p.M - 1) * p.lda;
#pragma unroll
  for (int i = 0; i < CB; ++i) pb[i] = p.B + (int64_t)min(n0 + (t >> 3) + i * (T / 8), p.N - 1) * p.ldb;
  const int c = t & 7;
  const int put = stage_byte(t >> 3, c);  // T/8 is a multiple of 16 rows: the same swizzle for every i
  static_assert((T / 8) % 16 == 0, "swizzle period");

  const float* sa[TM];
  const float* sb[BROW ? TN * 4 : TN];
#pragma unroll
  for (int j = 0; j < TM; ++j)
    sa[j] = p.SA + (int64_t)(min(m0 + (wm * TM + j) * 16 + r, p.M - 1) >> p.sa_sh) * p.sa_r;
#pragma unroll
  for (int i = 0; i < TN; ++i) {
    const int n = n0 + (wn * TN + i) * 16;
    if constexpr (BROW) {
#pragma unroll
      for (int e = 0; e < 4; ++e) sb[i * 4 + e] = p.SB + (int64_t)min(n + 4 * g + e, p.N - 1) * p.sb_r;
    } else {
      sb[i] = p.SB + (int64_t)(min(n, p.N - 1) >> 7) * p.sb_r;
    }
  }

  f32x4 acc[TM][TN];
#pragma unroll
  for (int j = 0; j < TM; ++j)
#pragma unroll
    for (int i = 0; i < TN; ++i) acc[j][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  u32x4_t ra[CA], rb[CB];
  auto load = [&](int kb) {
    const int k = kb * 128 + c * 16;
    if (kb * 128 + 128 <= p.K) {
#pragma unroll
      for (int i = 0; i < CA; ++i) ra[i] = *reinterpret_cast<const u32x4_a1*>(pa[i] + k);
#pragma unroll
      for (int i = 0; i < CB; ++i) rb[i] = *reinterpret_cast<const u32x4_a1*>(pb[i] + k);
    } else {
#pragma unroll
      for (int i = 0; i < CA; ++i) ra[i] = load_chunk(pa[i], k, p.K);
#pragma unroll
      for (int i = 0; i < CB; ++i) rb[i] = load_chunk(pb[i], k, p.K);
    }
  };
  auto store = [&](uint8_t* st) {
#pragma unroll
    for (int i = 0; i < CA; ++i) *reinterpret_cast<u32x4_t*>(st + put + i * T * 16) = ra[i];
#pragma unroll
    for (int i = 0; i < CB; ++i) *reinterpret_cast<u32x4_t*>(st + BM * 128 + put + i * T * 16) = rb[i];
  };
  load(0);
  store(smem[0]);
  __syncthreads();
  for (int kb = 0; kb < nkb; ++kb) {
    const uint8_t* st = smem[kb & 1];
    if (kb + 1 < nkb) load(kb + 1);
    float fa[TM], fb[BROW ? TN * 4 : TN];
#pragma unroll
    for (int j = 0; j < TM; ++j) fa[j] = sa[j][kb * p.sa_c];
#pragma unroll
    for (int i = 0; i < (BROW ? TN * 4 : TN); ++i) fb[i] = sb[i][kb * p.sb_c];
    Frag<BF, EXACT> b[TN];
#pragma unroll
    for (int i = 0; i < TN; ++i) b[i] = read_frag<BF, EXACT>(st + BM * 128, (wn * TN + i) * 16 + r, g);
#pragma unroll
    for (int j = 0; j < TM; ++j) {
      const Frag<AF, EXACT> a = read_frag<AF, EXACT>(st, (wm * TM + j) * 16 + r, g);
#pragma unroll
      for (int i = 0; i < TN; ++i) {
        const f32x4 d = mfma_block<AF, BF>(b[i], a);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[j][i][e] = fmaf(d[e], fa[j] * fb[BROW ? i * 4 + e : i], acc[j][i][e]);
      }
    }
    if (kb + 1 < nkb) store(smem[(kb + 1) & 1]);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < TN; ++i) {
    const int n = n0 + (wn * TN + i) * 16 + 4 * g, left = p.N - n;
    f32x4 bv = {0.0f, 0.0f, 0.0f, 0.0f};
    if (p.bias) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < left) bv[e] = p.bias[n + e];
    }
#pragma unroll
    for (int j = 0; j < TM; ++j) {
      const int m = m0 + (wm * TM + j) * 16 + r;
      if (m < p.M) store_out4(p.C, p.out, (int64_t)m * p.ldc + n, acc[j][i] + bv, left);
    }
  }
}

// ---------------------------------------------------------------------------
// Operands whose rows are 16-byte aligned: tiles go straight into LDS (a lane's
// 16 bytes at the place its swizzled chunk has), and so do the block's scales,
// one a lane; S stages, one barrier a block of K.  The barrier stands before the
// block's last row of fragments: there the wave has read all it needs of the
// stage, the next stage has landed, the loads of block kb + S go out into the
// freed stage, and the next fragments are read under the remaining products.  A
// block's results are added to the accumulators one row of fragments late, so
// that no multiply-add waits for its MFMA.  A last, partial block goes through
// registers with zeros behind K.
// 8192 x 4096 x 4096 bf16 126-138 us (2.0-2.2 PFLOP/s; the library's 8-bit product
// 2.8): by its counters the matrix cores are busy 47% of the cycles (at 2.07 GHz),
// the other VALU instructions, 5.5 an MFMA, take 33% at 4 cycles each, the waves wait
// for loads, LDS or the barrier in 31% of their time, and 11% of the cycles a CU
// has no wave (it takes two tiles one after the other, one workgroup at a time, so
// each tile's first loads and its output stand alone).  Issue alone explains little of
// it: an 8-bit MFMA issues every 35 cycles a SIMD, with the 5 multiply-adds of a
// block's results every 39, with 8 (B's scales by rows) 49.
// 11008 x 4096 x 8192 f32 700 us (1.05; bf16 products 1.45): MFMA busy 50% of the
// cycles (at 1.83 GHz), the 4.3 other VALU instructions an MFMA 54%, so the two
// hardly overlap.  Two of those are conversions, one more than needed: each
// fragment is converted by the two waves that read it.  256 x 256 tiles would need
// their f32 output staged in parts; they were not tried so.
// 1 x 32000 x 4096 f32: 21-25 us, B at 5.2-6.1 TB/s.
// ---------------------------------------------------------------------------
template <int BM, int BN, int WM, int WN, int S, int AF, int BF, bool BROW, bool EXACT>
__global__ __launch_bounds__(64 * WM * WN, 2) void gemm_fp8_lds_kernel(Fp8Gemm p) {
  constexpr int T = 64 * WM * WN, NW = WM * WN;
  constexpr int TM = BM / WM / 16, TN = BN / WN / 16;
  constexpr int PA = BM / 8 / NW, PB = BN / 8 / NW;  // 1 KB loads a wave and stage
  constexpr int STAGE = (BM + BN) * 128;
  // scales: wave w fetches those of rows 64 w .. of the tile's A rows and then B
  // rows; waves beyond them repeat the last ones, so that every wave has the
  // same loads in flight
  constexpr int SBM = (BM + 63) / 64 * 64;  // (a tile of 32 rows: as for 64)
  constexpr int SW = (SBM + BN) / 64, NVM = PA + PB + 1;
  static_assert(SBM + BN <= T && BN % 64 == 0 && PA * NW * 8 == BM && PB * NW * 8 == BN,
                "whole loads a wave");
  static_assert(S >= 2 && (S - 1) * NVM < 64, "loads in flight are counted in 6 bits");
  __shared__ __attribute__((aligned(1024))) uint8_t smem[S * STAGE];
  __shared__ __attribute__((aligned(16))) float scales[S][64 * (SW < NW ? SW + 1 : SW)];
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int wm = wave / WN, wn = wave % WN, r = lane & 15, g = lane >> 4;
  int tile_m, tile_n;
  tile_coords_of(blockIdx.x, p.tiles_m, p.tiles_n, tile_m, tile_n);
  const int m0 = tile_m * BM, n0 = tile_n * BN;
  const int nfull = p.K >> 7;

  // loads: wave w fills the blocks of 8 rows w, w + NW, ... of each operand
  const int last_a = min(p.M - m0, BM) - 1, last_b = min(p.N - n0, BN) - 1;
  const i32x4_t rsrc_a = buffer_rsrc(p.A + (int64_t)m0 * p.lda, (uint32_t)(last_a * p.lda + p.K));
  const i32x4_t rsrc_b = buffer_rsrc(p.B + (int64_t)n0 * p.ldb, (uint32_t)(last_b * p.ldb + p.K));
  int va[PA], vb[PB];
#pragma unroll
  for (int i = 0; i < PA; ++i) {
    const int row = (wave + i * NW) * 8 + (lane >> 3);
    va[i] = min(row, last_a) * (int)p.lda + (((lane & 7) ^ ((row >> 1) & 7)) << 4);
  }
#pragma unroll
  for (int i = 0; i < PB; ++i) {
    const int row = (wave + i * NW) * 8 + (lane >> 3);
    vb[i] = min(row, last_b) * (int)p.ldb + (((lane & 7) ^ ((row >> 1) & 7)) << 4);
  }
  const bool of_a = wave < SBM / 64;
  const int srow = (of_a ? wave : min(wave - SBM / 64, BN / 64 - 1)) * 64 + lane;
  const int64_t s_first = of_a ? (int64_t)(m0 >> p.sa_sh) * p.sa_r : (int64_t)(n0 >> p.sb_sh) * p.sb_r;
  const i32x4_t rsrc_s = buffer_rsrc((of_a ? p.SA : p.SB) + s_first, 0x7fffffffu);
  const int s_step = of_a ? (int)p.sa_c * 4 : (int)p.sb_c * 4;
  const int vs = of_a ? (((m0 + min(srow, last_a)) >> p.sa_sh) - (m0 >> p.sa_sh)) * (int)p.sa_r * 4
                      : (((n0 + min(srow, last_b)) >> p.sb_sh) - (n0 >> p.sb_sh)) * (int)p.sb_r * 4;

  // (inline asm: the compiler would wait for all loads in flight before every
  // LDS read that follows one)
  auto issue = [&](int kb, auto pad) {
    constexpr bool PAD = decltype(pad)::value;
    const int slot = S == 2 ? kb & 1 : kb % S;
    const uint32_t st = (uint32_t)(uintptr_t)(smem + slot * STAGE);
#pragma unroll
    for (int i = 0; i < PA; ++i) asm_buffer_load_lds<PAD>(rsrc_a, st + (wave + i * NW) * 1024, va[i], kb * 128);
#pragma unroll
    for (int i = 0; i < PB; ++i)
      asm_buffer_load_lds<PAD>(rsrc_b, st + BM * 128 + (wave + i * NW) * 1024, vb[i], kb * 128);
    asm_buffer_load_lds4<PAD>(rsrc_s, (uint32_t)(uintptr_t)(scales[slot] + min(wave, SW) * 64), vs, kb * s_step);
  };
  // Waits for all but the last n blocks' loads of the wave, n < S - 1.
  auto wait_blocks = [&](int n) {
    if constexpr (S > 3)
      if (n >= 2) return wait_vm_lgkm0<2 * NVM>();
    if constexpr (S > 2)
      if (n == 1) return wait_vm_lgkm0<NVM>();
    wait_vm_lgkm0<0>();
    // the loads' offsets stay in their registers until the last load has landed
#pragma unroll
    for (int i = 0; i < PA; ++i) asm volatile("" ::"v"(va[i]));
#pragma unroll
    for (int i = 0; i < PB; ++i) asm volatile("" ::"v"(vb[i]));
    asm volatile("" ::"v"(vs));
  };
  static_assert(S <= 4, "wait_blocks");

  f32x4 acc[TM][TN];
#pragma unroll
  for (int j = 0; j < TM; ++j)
#pragma unroll
    for (int i = 0; i < TN; ++i) acc[j][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  Frag<BF, EXACT> b[TN];
  Frag<AF, EXACT> a;
  const int row_a = wm * TM * 16 + r, row_b = wn * TN * 16 + r;
  auto read_a = [&](const uint8_t* st, int j) { return read_frag<AF, EXACT>(st, row_a + j * 16, g); };
  auto read_b = [&](const uint8_t* st, int i) { return read_frag<BF, EXACT>(st + BM * 128, row_b + i * 16, g); };

  auto stage_of = [&](int kb) { return S == 2 ? kb & 1 : kb % S; };
  // One block.  MODE 0: the last one; 1: the next stage is read on into; 2: and
  // the loads of block kb + S go out.
  auto block = [&](int kb, auto mode) {
    constexpr int MODE = decltype(mode)::value;
    constexpr bool NEXT = MODE > 0;
    const uint8_t* st = smem + stage_of(kb) * STAGE;
    const float* sl = scales[stage_of(kb)];
    // by blocks, the wave's columns (at most 128, and no block's end among
    // them) share one scale
    static_assert(128 % (TN * 16) == 0, "a wave's columns lie in one block");
    float fb[BROW ? TN * 4 : 1];
    if constexpr (BROW) {
#pragma unroll
      for (int i = 0; i < TN; ++i) {
        const f32x4 v = *reinterpret_cast<const f32x4*>(sl + SBM + (wn * TN + i) * 16 + 4 * g);
#pragma unroll
        for (int e = 0; e < 4; ++e) fb[i * 4 + e] = v[e];
      }
    } else {
      fb[0] = sl[SBM + wn * TN * 16];
    }
    f32x4 d[2][TN];
    float fa[2];
    auto add = [&](int j) {
#pragma unroll
      for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          acc[j][i][e] = fmaf(d[j & 1][i][e], fa[j & 1] * fb[BROW ? i * 4 + e : 0], acc[j][i][e]);
    };
#pragma unroll
    for (int j = 0; j < TM; ++j) {
      fa[j & 1] = sl[row_a + j * 16];
      Frag<AF, EXACT> an;
      if (j + 1 < TM) {
        an = read_a(st, j + 1);
      } else if constexpr (NEXT) {
        if constexpr (MODE == 2) wait_vm_lgkm0<(S - 2) * NVM>();
        else wait_blocks(nfull - 2 - kb);
        barrier_keep_loads();
        if constexpr (MODE == 2) issue(kb + S, std::false_type{});
        an = read_a(smem + stage_of(kb + 1) * STAGE, 0);
      }
#pragma unroll
      for (int i = 0; i < TN; ++i) d[j & 1][i] = mfma_block<AF, BF>(b[i], a);
      if (j > 0) add(j - 1);
      if (j + 1 == TM) {
        if constexpr (NEXT) {
#pragma unroll
          for (int i = 0; i < TN; ++i) b[i] = read_b(smem + stage_of(kb + 1) * STAGE, i);
        }
      }
      if (j + 1 < TM || NEXT) a = an;
      if (!EXACT && j > 0 && j + 1 < TM) {  // the multiply-adds of row j - 1 between the MFMAs of row j
        __builtin_amdgcn_sched_group_barrier(0x100, 3, 0);
#pragma unroll
        for (int i = 0; i < TN; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x002, BROW ? 8 : 5, 0);
        }
      }
      __builtin_amdgcn_sched_barrier(0);  // a row of fragments at a time: more at once would spill
    }
    add(TM - 1);
  };

  // nfull >= 2
  issue(0, std::true_type{});
  if constexpr (S > 2) {
    for (int q = 1; q < S - 1 && q < nfull; ++q) issue(q, std::true_type{});
    wait_blocks(min(nfull - 1, S - 2));
  } else {
    wait_blocks(0);
  }
  barrier_keep_loads();
  if (S == 2 || S - 1 < nfull) issue(S - 1, std::true_type{});
#pragma unroll
  for (int i = 0; i < TN; ++i) b[i] = read_b(smem, i);
  a = read_a(smem, 0);
  int kb = 0;
  for (; kb + S < nfull; ++kb) block(kb, std::integral_constant<int, 2>{});
  for (; kb + 1 < nfull; ++kb) block(kb, std::integral_constant<int, 1>{});
  block(kb, std::integral_constant<int, 0>{});
  if (p.K & 127) {
    __syncthreads();
    uint8_t* st = smem + stage_of(nfull) * STAGE;
    const int c = t & 7;
#pragma unroll 1
    for (int row = t >> 3; row < BM; row += T / 8)
      *reinterpret_cast<u32x4_t*>(st + stage_byte(row, c)) =
          load_chunk(p.A + (int64_t)min(m0 + row, p.M - 1) * p.lda, nfull * 128 + c * 16, p.K);
#pragma unroll 1
    for (int row = t >> 3; row < BN; row += T / 8)
      *reinterpret_cast<u32x4_t*>(st + BM * 128 + stage_byte(row, c)) =
          load_chunk(p.B + (int64_t)min(n0 + row, p.N - 1) * p.ldb, nfull * 128 + c * 16, p.K);
    if (t < SBM + BN) {
      const bool ra = t < SBM;
      scales[stage_of(nfull)][t] =
          ra ? p.SA[(int64_t)((m0 + min(t, last_a)) >> p.sa_sh) * p.sa_r + nfull * p.sa_c]
             : p.SB[(int64_t)((n0 + min(t - SBM, last_b)) >> p.sb_sh) * p.sb_r + nfull * p.sb_c];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < TN; ++i) b[i] = read_b(st, i);
    a = read_a(st, 0);
    block(nfull, std::integral_constant<int, 0>{});
  }

  // The tile goes through LDS, so that whole rows are stored, 16 bytes a lane:
  // chunk c of a row at c ^ (row mod the row's chunks).
  constexpr int OB = EXACT ? 4 : 2, ROWB = BN * OB, CPR = ROWB / 16, EPC = 16 / OB;
  static_assert(BM * ROWB <= S * STAGE && BM * CPR % T == 0, "the tile fits the stages");
  __syncthreads();
#pragma unroll
  for (int i = 0; i < TN; ++i) {
    const int nl = (wn * TN + i) * 16 + 4 * g, left = p.N - n0 - nl;
    f32x4 bv = {0.0f, 0.0f, 0.0f, 0.0f};
    if (p.bias) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < left) bv[e] = p.bias[n0 + nl + e];
    }
#pragma unroll
    for (int j = 0; j < TM; ++j) {
      const int row = row_a + j * 16;
      const f32x4 v = acc[j][i] + bv;
      uint8_t* at = smem + row * ROWB + (((nl / EPC) ^ (row & (CPR - 1))) << 4);
      if constexpr (EXACT) *reinterpret_cast<f32x4*>(at) = v;
      else *reinterpret_cast<uint2*>(at + (nl & 4) * 2) = pack_out4(p.out, v);
    }
  }
  __syncthreads();
#pragma unroll 4
  for (int q = t; q < BM * CPR; q += T) {
    const int row = q / CPR, c = q % CPR, n = n0 + c * EPC;
    const u32x4_t v = *reinterpret_cast<const u32x4_t*>(smem + row * ROWB + ((c ^ (row & (CPR - 1))) << 4));
    if (m0 + row >= p.M || n >= p.N) continue;
    uint8_t* dst = static_cast<uint8_t*>(p.C) + ((int64_t)(m0 + row) * p.ldc + n) * OB;
    if (n + EPC <= p.N) {
      *reinterpret_cast<u32x4_a1*>(dst) = v;
    } else {
#pragma unroll
      for (int e = 0; e < EPC - 1; ++e)
        if (n + e < p.N) {
          if constexpr (EXACT) reinterpret_cast<uint32_t*>(dst)[e] = v[e];
          else reinterpret_cast<uint16_t*>(dst)[e] = (uint16_t)(v[e >> 1] >> (16 * (e & 1)));
        }
    }
  }
}

// ---------------------------------------------------------------------------
// At most 16 TM rows of A: the bytes of B are what counts.  A wave takes 16
// rows of B over a share of K, straight into registers (a row's 128 bytes of a
// block are one cache line), the KW waves of a workgroup share K and add up
// through LDS in a fixed order.  Any alignment.  Products and sums in f32, as
// for f32 outputs above: the matrix cores have nothing else to do.  1 x 4096 x
// 4096 4.9 us, 16 rows 7.0: one round of loads and the sum over the waves; beyond
// two workgroups a CU each repeats that, and A's rows (1 x 11008 x 4096 13.3).
// ---------------------------------------------------------------------------
template <int TM, int KW, int AF, int BF, bool BROW>
__global__ __launch_bounds__(64 * KW) void gemm_fp8_rows_kernel(Fp8Gemm p) {
  constexpr int U = TM == 1 ? 4 : 2;  // blocks in flight
  __shared__ __attribute__((aligned(16))) f32x4 part[KW][TM][64];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, r = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const int nkb = (p.K + 127) >> 7;
  const int k0 = (int)((int64_t)nkb * wave / KW), k1 = (int)((int64_t)nkb * (wave + 1) / KW);
  const uint8_t* pb = p.B + (int64_t)min(n0 + r, p.N - 1) * p.ldb;
  const uint8_t* pa[TM];
  const float* sa[TM];
#pragma unroll
  for (int j = 0; j < TM; ++j) {
    const int m = min(j * 16 + r, p.M - 1);
    pa[j] = p.A + (int64_t)m * p.lda;
    sa[j] = p.SA + (int64_t)(m >> p.sa_sh) * p.sa_r;
  }
  const float* sb[BROW ? 4 : 1];
#pragma unroll
  for (int e = 0; e < (BROW ? 4 : 1); ++e)
    sb[e] = p.SB + (int64_t)(min(n0 + (BROW ? 4 * g + e : 0), p.N - 1) >> p.sb_sh) * p.sb_r;

  f32x4 acc[TM];
#pragma unroll
  for (int j = 0; j < TM; ++j) acc[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  auto add = [&](int kb, const Frag<BF, true>& b, const Frag<AF, true>& a, int j, const float (&fb)[BROW ? 4 : 1],
                 float fa) {
    const f32x4 d = mfma_block<AF, BF>(b, a);
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[j][e] = fmaf(d[e], fa * fb[BROW ? e : 0], acc[j][e]);
  };
  // 32 bytes a lane of a row: whole (WHOLE) or up to K
  auto frag = [&](auto& f, const uint8_t* row, int kb, auto whole) {
    const int k = kb * 128 + g * 16;
    if constexpr (decltype(whole)::value)
      f.set(*reinterpret_cast<const u32x4_a1*>(row + k), *reinterpret_cast<const u32x4_a1*>(row + k + 64));
    else
      f.set(load_chunk(row, k, p.K), load_chunk(row, k + 64, p.K));
  };
  auto one = [&](int kb, auto whole) {
    Frag<BF, true> b;
    frag(b, pb, kb, whole);
    float fb[BROW ? 4 : 1];
#pragma unroll
    for (int e = 0; e < (BROW ? 4 : 1); ++e) fb[e] = sb[e][kb * p.sb_c];
#pragma unroll
    for (int j = 0; j < TM; ++j) {
      Frag<AF, true> a;
      frag(a, pa[j], kb, whole);
      add(kb, b, a, j, fb, sa[j][kb * p.sa_c]);
    }
  };
  const int kw = min(k1, p.K >> 7);  // whole blocks
  int kb = k0;
  for (; kb + U <= kw; kb += U) {
    u32x4_t wb[U][2], wa[U][TM][2];
    float fb[U][BROW ? 4 : 1], fa[U][TM];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = (kb + u) * 128 + g * 16;
      wb[u][0] = *reinterpret_cast<const u32x4_a1*>(pb + k);
      wb[u][1] = *reinterpret_cast<const u32x4_a1*>(pb + k + 64);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = (kb + u) * 128 + g * 16;
#pragma unroll
      for (int j = 0; j < TM; ++j) {
        wa[u][j][0] = *reinterpret_cast<const u32x4_a1*>(pa[j] + k);
        wa[u][j][1] = *reinterpret_cast<const u32x4_a1*>(pa[j] + k + 64);
        fa[u][j] = sa[j][(kb + u) * p.sa_c];
      }
#pragma unroll
      for (int e = 0; e < (BROW ? 4 : 1); ++e) fb[u][e] = sb[e][(kb + u) * p.sb_c];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      Frag<BF, true> b;
      b.set(wb[u][0], wb[u][1]);
#pragma unroll
      for (int j = 0; j < TM; ++j) {
        Frag<AF, true> a;
        a.set(wa[u][j][0], wa[u][j][1]);
        add(kb + u, b, a, j, fb[u], fa[u][j]);
      }
    }
  }
  for (; kb < kw; ++kb) one(kb, std::true_type{});
  if (kb < k1) one(kb, std::false_type{});  // the last, partial block

#pragma unroll
  for (int j = 0; j < TM; ++j) part[wave][j][lane] = acc[j];
  __syncthreads();
  if (wave < TM) {  // wave j adds up and stores the j-th 16 rows
    f32x4 v = part[0][wave][lane];
#pragma unroll
    for (int w = 1; w < KW; ++w) v = v + part[w][wave][lane];
    const int m = wave * 16 + r, n = n0 + 4 * g, left = p.N - n;
    if (p.bias) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < left) v[e] += p.bias[n + e];
    }
    if (m < p.M) store_out4(p.C, p.out, (int64_t)m * p.ldc + n, v, left);
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
// Scales of a [rows, cols] operand: by rows or by blocks, any strides.
bool scale_in(const TensorDesc& t, int64_t rows, int64_t cols, int* sh) {
  if (dt(t) != DType::kF32 || t.rank != 2 || t.shape[1] != (cols + 127) / 128) return false;
  if (t.stride[0] < 0 || t.stride[1] < 0) return false;
  if (t.shape[0] == rows) *sh = 0;
  else if (t.shape[0] == (rows + 127) / 128) *sh = 7;
  else return false;
  return true;
}

bool gemm_fp8_sup(const TensorDesc* in, int ni, const TensorDesc* out, int no, const void*) {
  if (!in || !out || (ni != 4 && ni != 5) || no != 1) return false;
  int64_t lda, ldb, ldc;
  int sh, ek;
  if (!is_fp8(in[0]) || !is_fp8(in[2]) || !matrix_ld(in[0], false, &lda) || !matrix_ld(in[2], false, &ldb))
    return false;
  const int64_t M = in[0].shape[0], K = in[0].shape[1], N = in[2].shape[0];
  constexpr int64_t kMax = (int64_t{1} << 31) - 512;
  if (K < 1 || in[2].shape[1] != K || M > kMax || N > kMax || K > kMax) return false;
  if (!scale_in(in[1], M, K, &sh) || !scale_in(in[3], N, K, &sh)) return false;
  if (ni == 5 && !vector_of(in[4], DType::kF32, N)) return false;
  if (!elem_kind(out[0], &ek) || !matrix_ld(out[0], true, &ldc)) return false;
  if (out[0].shape[0] != M || out[0].shape[1] != N) return false;
  return !any_overlap(in, ni, out, no);
}

// S: stages of the kernel that loads straight into LDS; 0: the one of any
// alignment.  EXACT: f32 outputs.
template <int S, bool EXACT, int BM, int BN, int WM, int WN, int AF, int BF>
Status run_tiles(Fp8Gemm& p, hipStream_t s) {
  p.tiles_m = (p.M + BM - 1) / BM;
  p.tiles_n = (p.N + BN - 1) / BN;
  constexpr int T = 64 * WM * WN;
  const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n;
  if (tiles * T > UINT32_MAX) return Status::InvalidArgument;  // a grid's lanes are counted in 32 bits
  const unsigned g = (unsigned)tiles;
  auto go = [&](auto brow) {
    constexpr bool R = decltype(brow)::value;
    if constexpr (S > 0) gemm_fp8_lds_kernel<BM, BN, WM, WN, S, AF, BF, R, EXACT><<<g, T, 0, s>>>(p);
    else gemm_fp8_kernel<BM, BN, WM, WN, AF, BF, R, EXACT><<<g, T, 0, s>>>(p);
  };
  if (p.sb_sh == 0) go(std::true_type{});
  else go(std::false_type{});
  return launch_status("gemm_fp8");
}

template <int AF, int BF>
Status gemm_fp8_run(Fp8Gemm& p, hipStream_t s) {
  // straight into LDS: 16-byte aligned rows, a tile's bytes and scales within
  // 32-bit offsets, two blocks of K at least
  const int64_t nkb = (p.K + 127) / 128, lim = 1 << 22;
  const bool lds = aligned(p.A, 16) && aligned(p.B, 16) && p.lda % 16 == 0 && p.ldb % 16 == 0 && p.lda < lim &&
                   p.ldb < lim && p.sa_r < (lim >> 2) && p.sb_r < (lim >> 2) && nkb * p.sa_c < (1 << 26) &&
                   nkb * p.sb_c < (1 << 26) && p.K >= 256;
  if (p.M <= 32) {
    // Few columns: workgroups of 16 (or where tiles do not go straight into LDS).
    // From about two of those a CU on the tiles are the faster ones: 1 x 4096 x
    // 4096 4.9 us (tiles 8.8), 32 x 4096 x 4096 f32 9.6 (11.7), 16 x 8192 x 4096
    // f32 11.3 (11.6), 1 x 11008 x 4096 13.3 (9.0), 1 x 32000 x 4096 f32 32.1
    // (21.3), 32 rows 58.8 (21.4).
    const unsigned g = (unsigned)(((int64_t)p.N + 15) / 16);
    const int64_t work = (int64_t)g * (p.M <= 16 ? 1 : 2);
    if (lds && work > 512) {
      if (p.out == EL_F32) return run_tiles<4, true, 32, 64, 2, 2, AF, BF>(p, s);
      return run_tiles<4, false, 32, 64, 2, 2, AF, BF>(p, s);
    }
    if ((int64_t)g * 512 > UINT32_MAX) return Status::InvalidArgument;
    auto go = [&](auto tm) {
      constexpr int TM = decltype(tm)::value;
      if (p.sb_sh == 0) gemm_fp8_rows_kernel<TM, 8, AF, BF, true><<<g, 512, 0, s>>>(p);
      else gemm_fp8_rows_kernel<TM, 8, AF, BF, false><<<g, 512, 0, s>>>(p);
    };
    if (p.M <= 16) go(std::integral_constant<int, 1>{});
    else go(std::integral_constant<int, 2>{});
    return launch_status("gemm_fp8");
  }
  // Larger tiles where they fill the chip.  64 x 64 against 128 x 128: 256 x 4096
  // x 4096 bf16 11.5 us (22.0), 512 19.9 (24.0), 1024 32.9 (26.9); 1001 x 1003 x
  // 784 f16 6.6 (11.3).  128 x 128 against 256 x 256: 2048 x 4096 x 4096 40.2
  // (53.6), 4096 78.1 (63.4).
  auto tiles = [&](int64_t b) { return ((p.M + b - 1) / b) * ((p.N + b - 1) / b); };
  if (p.out == EL_F32) {
    if (!lds && tiles(128) < 256) return run_tiles<0, true, 64, 64, 2, 2, AF, BF>(p, s);
    if (!lds) return run_tiles<0, true, 128, 128, 2, 2, AF, BF>(p, s);
    if (tiles(128) < 256) return run_tiles<4, true, 64, 64, 2, 2, AF, BF>(p, s);
    return run_tiles<2, true, 128, 128, 2, 2, AF, BF>(p, s);
  }
  if (!lds && tiles(128) < 256) return run_tiles<0, false, 64, 64, 2, 2, AF, BF>(p, s);
  if (!lds) return run_tiles<0, false, 128, 128, 2, 2, AF, BF>(p, s);
  if (tiles(128) < 256) return run_tiles<4, false, 64, 64, 2, 2, AF, BF>(p, s);
  if (tiles(256) < 256) return run_tiles<2, false, 128, 128, 2, 2, AF, BF>(p, s);
  return run_tiles<2, false, 256, 256, 2, 4, AF, BF>(p, s);
}

Status gemm_fp8_launch(const TensorDesc* in, int ni, TensorDesc* out, int no, const void* at, void*, size_t,
                       void* stream) {
  if (!gemm_fp8_sup(in, ni, out, no, at)) return Status::InvalidArgument;
  if (numel_of(out[0]) == 0) return Status::Ok;
  for (int k = 0; k < ni; ++k)
    if (no_memory(in[k])) return Status::InvalidArgument;
  if (no_memory(out[0])) return Status::InvalidArgument;
  Fp8Gemm p{};
  p.A = (const uint8_t*)in[0].data;
  p.SA = (const float*)in[1].data;
  p.B = (const uint8_t*)in[2].data;
  p.SB = (const float*)in[3].data;
  p.bias = ni == 5 ? (const float*)in[4].data : nullptr;
  p.C = out[0].data;
  matrix_ld(in[0], false, &p.lda);
  matrix_ld(in[2], false, &p.ldb);
  matrix_ld(out[0], true, &p.ldc);
  p.sa_r = in[1].stride[0];
  p.sa_c = in[1].stride[1];
  p.sb_r = in[3].stride[0];
  p.sb_c = in[3].stride[1];
  p.M = (int)in[0].shape[0];
  p.K = (int)in[0].shape[1];
  p.N = (int)in[2].shape[0];
  scale_in(in[1], p.M, p.K, &p.sa_sh);
  scale_in(in[3], p.N, p.K, &p.sb_sh);
  elem_kind(out[0], &p.out);
  hipStream_t s = as_stream(stream);
  const bool a5 = dt(in[0]) == DType::kF8E5M2, b5 = dt(in[2]) == DType::kF8E5M2;
  if (a5) return b5 ? gemm_fp8_run<1, 1>(p, s) : gemm_fp8_run<1, 0>(p, s);
  return b5 ? gemm_fp8_run<0, 1>(p, s) : gemm_fp8_run<0, 0>(p, s);
}

size_t no_workspace(const TensorDesc*, int, const void*) { return 0; }

}  // namespace

KernelVariant make_gemm_fp8_variant() {
  KernelVariant v;
  v.name = "gemm_fp8";
  v.launch = gemm_fp8_launch;
  v.supported = gemm_fp8_sup;
  v.query_workspace = no_workspace;
  return v;
}

}  // namespace aicf::hip
