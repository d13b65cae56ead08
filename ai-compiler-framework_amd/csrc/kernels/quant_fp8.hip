// Matrices in 8-bit floating point with a scale for each block of 128.
//
//   X [M, K] f32/f16/bf16 -> Q [M, K] f8 (e4m3 or e5m2), S f32
//     by rows:   S [M, ceil(K/128)], one scale for 128 columns of a row
//     by blocks: S [ceil(M/128), ceil(K/128)], one for 128 x 128 elements
//   and, with four outputs, QT [K, M] and ST: the same of X^T, the operand of
//   the products that contract over X's rows (weight gradients of activations
//   and gradients, input gradients of weights).
//
//   s = max(amax / FMAX, 2^-126), FMAX = 448 (e4m3) or 57344 (e5m2); with bit 0
//   of the flags s is rounded up to a power of two.  q = x * (1 / s), rounded to
//   nearest even.  |x| <= amax gives |q| <= FMAX (1 + 3 * 2^-24), which rounds
//   to FMAX: no clamp is needed.  The power-of-two scales make x * (1 / s)
//   exact, so the codes are x / s rounded once.  Division and multiplication are
//   IEEE f32; amax is taken on the bits of |x|, where a NaN is above all numbers
//   and reaches its block's scale and codes.
//
// No counterpart in the reference.
#include "../common/head_util.hpp"

#include <type_traits>

namespace aicf::hip {

namespace {

constexpr int kB = 128;  // elements of a scale's block along a row

struct QuantArgs {
  const void* x;
  uint8_t* q;
  uint8_t* qt;
  float* s;
  float* st;
  int64_t M, K, ldx, ldq, ldqt;
  int64_t s_r, s_c, st_r, st_c;  // strides of S and ST
  int by_rows, pow2;
};

template <int F>
__device__ __forceinline__ float block_scale(uint32_t amax_bits, int pow2) {
  constexpr float FMAX = F == 0 ? 448.0f : 57344.0f;
  constexpr float MIN = 1.17549435e-38f;  // 2^-126
  float s = __uint_as_float(amax_bits) / FMAX;
  s = s < MIN ? MIN : s;  // a NaN stays
  if (pow2 && s == s) s = __uint_as_float((__float_as_uint(s) + 0x7fffffu) & 0x7f800000u);
  return s;
}

template <int F>
__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
  int w = 0;
  if constexpr (F == 0) {
    w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, w, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
  } else {
    w = __builtin_amdgcn_cvt_pk_bf8_f32(a, b, w, false);
    w = __builtin_amdgcn_cvt_pk_bf8_f32(c, d, w, true);
  }
  return (uint32_t)w;
}

__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// w (8 codes) to p[0 .. n).
__device__ __forceinline__ void store8(uint8_t* p, uint2 w, int64_t n) {
  if (n >= 8) {
    *reinterpret_cast<u32x2_a1*>(p) = u32x2_a1{w.x, w.y};
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) p[e] = (uint8_t)((e < 4 ? w.x : w.y) >> (8 * (e & 3)));
  }
}

// ---------------------------------------------------------------------------
// By rows, no transpose: 16 lanes hold a block (8 elements each), a wave 512
// columns of a row.  One read and one write of memory: 8192 x 4096 bf16 20.8 us
// (4.85 TB/s), f32 25.0 (6.7, from the cache), 16 x 4096 2.8.
// ---------------------------------------------------------------------------
template <int EK, int F>
__global__ __launch_bounds__(256) void quant_rows_kernel(QuantArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t per_row = (a.K + 511) / 512, units = a.M * per_row;
  const int64_t waves = (int64_t)gridDim.x * 4;
  for (int64_t u = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); u < units; u += waves) {
    const int64_t row = u / per_row, c = (u % per_row) * 512 + lane * 8;
    float v[8];
    load8<EK>(v, a.x, row * a.ldx + c, a.K - c);
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) m = max(m, abs_bits(v[e]));
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, off, 64));
    const float s = block_scale<F>(m, a.pow2), inv = 1.0f / s;
    if (c >= a.K) continue;
    if ((lane & 15) == 0) a.s[row * a.s_r + (c / kB) * a.s_c] = s;
    const uint2 w{pack4<F>(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv),
                  pack4<F>(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv)};
    store8(a.q + row * a.ldq + c, w, a.K - c);
  }
}

// ---------------------------------------------------------------------------
// A 128 x 128 tile a workgroup, in registers: thread (tr, tc) holds rows
// 8 tr .. +7 and columns 8 tc .. +7.  Row maxima are taken over the 16 lanes of
// a row's threads, column maxima through LDS; then each thread makes one of the
// 256 scales (two IEEE divisions: 8 + 8 of them in every thread were half of
// this kernel's time).  The transposed codes go through LDS in pieces of 8 (one
// column's 8 rows), piece tr of column c at tr ^ (c >> 3).
// 8192 x 4096 bf16 by rows both ways 24.0 us (5.7 TB/s), 11008 x 4096 f32 by blocks
// both ways 44.3 (6.1): HBM.
// ---------------------------------------------------------------------------
// max over the 16 lanes of a DPP row
__device__ __forceinline__ uint32_t row16_max(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xf, 0xf, false));  // row_ror:8
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xf, 0xf, false));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x122, 0xf, 0xf, false));
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x121, 0xf, 0xf, false));
}

// EDGE: M or K has a last block that is not full.  ROWS: scales by rows (with a
// transpose).  TRANS: with a transpose.
template <int EK, int F, bool EDGE, bool ROWS, bool TRANS>
__global__ __launch_bounds__(256, 3) void quant_tile_kernel(QuantArgs a) {
  typedef uint32_t u32x4v __attribute__((ext_vector_type(4)));
  __shared__ __attribute__((aligned(16))) uint32_t cmax[16][kB];  // [tr][column]
  __shared__ __attribute__((aligned(16))) uint32_t rmax[kB];
  __shared__ __attribute__((aligned(16))) float inv_c[kB], inv_r[kB];
  __shared__ __attribute__((aligned(16))) uint8_t tile[kB * kB];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int tr = t >> 4, tc = t & 15;
  const uint32_t tiles_k = (uint32_t)((a.K + kB - 1) / kB);
  const int64_t tm = blockIdx.x / tiles_k, tk = blockIdx.x % tiles_k;
  const int64_t r0 = tm * kB + tr * 8, c0 = tk * kB + tc * 8;
  const int64_t nc = a.K - c0, nr = a.M - r0;
  const bool whole = !EDGE || (tm * kB + kB <= a.M && tk * kB + kB <= a.K);  // uniform
  float v[8][8];
  if (whole) {
#pragma unroll
    for (int i = 0; i < 8; ++i) load8<EK>(v[i], a.x, (r0 + i) * a.ldx + c0, 8);
  } else {  // past an edge: the last row or column again, and zeros in its place
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t at = (i < nr ? r0 + i : a.M - 1) * a.ldx;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float x = elem_f32<EK>(a.x, at + (j < nc ? c0 + j : a.K - 1));
        v[i][j] = i < nr && j < nc ? x : 0.0f;
      }
      __builtin_amdgcn_sched_barrier(0);  // a row's addresses at a time
    }
  }

  uint32_t rm[8], cm[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) rm[e] = cm[e] = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t b = abs_bits(v[i][j]);
      rm[i] = max(rm[i], b);
      cm[j] = max(cm[j], b);
    }
  if constexpr (!ROWS) {
    uint32_t b = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) b = max(b, cm[j]);
    b = row16_max(b);
    b = max(b, (uint32_t)__shfl_xor((int)b, 16, 64));
    b = max(b, (uint32_t)__shfl_xor((int)b, 32, 64));
    if (lane == 0) rmax[wave] = b;
    __syncthreads();
    const float s = block_scale<F>(max(max(rmax[0], rmax[1]), max(rmax[2], rmax[3])), a.pow2);
    if (t < kB) inv_r[t] = 1.0f / s;
    else inv_c[t - kB] = 1.0f / s;
    if (t == 0) {
      a.s[tm * a.s_r + tk * a.s_c] = s;
      if (TRANS) a.st[tk * a.st_r + tm * a.st_c] = s;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) rm[i] = row16_max(rm[i]);
    if (tc == 0) {
      *reinterpret_cast<u32x4v*>(&rmax[tr * 8]) = u32x4v{rm[0], rm[1], rm[2], rm[3]};
      *reinterpret_cast<u32x4v*>(&rmax[tr * 8 + 4]) = u32x4v{rm[4], rm[5], rm[6], rm[7]};
    }
    if constexpr (TRANS) {
      *reinterpret_cast<u32x4v*>(&cmax[tr][tc * 8]) = u32x4v{cm[0], cm[1], cm[2], cm[3]};
      *reinterpret_cast<u32x4v*>(&cmax[tr][tc * 8 + 4]) = u32x4v{cm[4], cm[5], cm[6], cm[7]};
    }
    __syncthreads();
    if (t < kB) {
      const float s = block_scale<F>(rmax[t], a.pow2);
      inv_r[t] = 1.0f / s;
      if (tm * kB + t < a.M) a.s[(tm * kB + t) * a.s_r + tk * a.s_c] = s;
    } else {
      const int c = t - kB;
      uint32_t b = 0;
#pragma unroll
      for (int i = 0; i < 16; ++i) b = max(b, cmax[i][c]);
      const float s = block_scale<F>(b, a.pow2);
      inv_c[c] = 1.0f / s;
      if (tk * kB + c < a.K) a.st[(tk * kB + c) * a.st_r + tm * a.st_c] = s;
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float r = inv_r[tr * 8 + i];
    const uint2 w{pack4<F>(v[i][0] * r, v[i][1] * r, v[i][2] * r, v[i][3] * r),
                  pack4<F>(v[i][4] * r, v[i][5] * r, v[i][6] * r, v[i][7] * r)};
    if (whole) store8(a.q + (r0 + i) * a.ldq + c0, w, 8);
    else if (i < nr) store8(a.q + (r0 + i) * a.ldq + c0, w, nc);
  }
  if constexpr (TRANS) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float r = inv_c[tc * 8 + j];
      const uint2 w{pack4<F>(v[0][j] * r, v[1][j] * r, v[2][j] * r, v[3][j] * r),
                    pack4<F>(v[4][j] * r, v[5][j] * r, v[6][j] * r, v[7][j] * r)};
      *reinterpret_cast<uint2*>(tile + (tc * 8 + j) * kB + ((tr ^ tc) * 8)) = w;
    }
    __syncthreads();
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const int c = p * 32 + (t >> 3), piece = (t & 7) * 2, f = c >> 3;
      const uint2 lo = *reinterpret_cast<const uint2*>(tile + c * kB + ((piece ^ f) * 8));
      const uint2 hi = *reinterpret_cast<const uint2*>(tile + c * kB + (((piece + 1) ^ f) * 8));
      const int64_t k = tk * kB + c, m = tm * kB + piece * 8, n = a.M - m;
      if (k < a.K) {
        uint8_t* dst = a.qt + k * a.ldqt + m;
        if (n >= 16) {
          *reinterpret_cast<u32x4_a1*>(dst) = u32x4_a1{lo.x, lo.y, hi.x, hi.y};
        } else {
          store8(dst, lo, n);
          store8(dst + 8, hi, n - 8);
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
int64_t blocks_of(int64_t n) { return (n + kB - 1) / kB; }

// Strides of a scale matrix an op writes: row-major or column-major.
bool scale_out(const TensorDesc& t, int64_t* r, int64_t* c) {
  if (dt(t) != DType::kF32 || t.rank != 2) return false;
  *r = t.stride[0];
  *c = t.stride[1];
  if (t.shape[0] <= 1 && t.shape[1] <= 1) return true;
  if (t.shape[0] <= 1) return *c >= 1;
  if (t.shape[1] <= 1) return *r >= 1;
  return (*c == 1 && *r >= t.shape[1]) || (*r == 1 && *c >= t.shape[0]);
}

bool quant_sup(const TensorDesc* in, int ni, const TensorDesc* out, int no, const void* attr) {
  if (!in || !out || ni != 1 || (no != 2 && no != 4)) return false;
  const AttrBlob& b = blob(attr);
  if (b.schema_id == AICF_SCHEMA_QFP8 && (!payload_ok(b, 4) || (field<int32_t>(b, 0) & ~1))) return false;
  int ek;
  int64_t ld, r, c;
  if (!elem_kind(in[0], &ek) || !matrix_ld(in[0], false, &ld)) return false;
  const int64_t M = in[0].shape[0], K = in[0].shape[1];
  if (K < 1 || blocks_of(M) * blocks_of(K) >= 1 << 24) return false;  // a grid's lanes are counted in 32 bits
  bool may_rows = true, may_blocks = true;
  for (int k = 0; k < no; k += 2) {
    const int64_t R = k ? K : M, C = k ? M : K;
    if (!is_fp8(out[k]) || out[k].dtype != out[0].dtype || !matrix_ld(out[k], true, &ld)) return false;
    if (out[k].shape[0] != R || out[k].shape[1] != C) return false;
    if (!scale_out(out[k + 1], &r, &c) || out[k + 1].shape[1] != blocks_of(C)) return false;
    may_rows = may_rows && out[k + 1].shape[0] == R;
    may_blocks = may_blocks && out[k + 1].shape[0] == blocks_of(R);
  }
  return (may_rows || may_blocks) && !any_overlap(in, ni, out, no);
}

template <int EK, int F>
Status quant_run(const QuantArgs& a, hipStream_t s) {
  if (a.by_rows && !a.qt) {
    const int64_t waves = a.M * ((a.K + 511) / 512);
    quant_rows_kernel<EK, F><<<grid_1d(waves, 4, 1 << 20), 256, 0, s>>>(a);
  } else {
    const unsigned g = (unsigned)(blocks_of(a.M) * blocks_of(a.K));
    auto go = [&](auto rows, auto trans) {
      constexpr bool R = decltype(rows)::value, T = decltype(trans)::value;
      if (a.M % kB || a.K % kB) quant_tile_kernel<EK, F, true, R, T><<<g, 256, 0, s>>>(a);
      else quant_tile_kernel<EK, F, false, R, T><<<g, 256, 0, s>>>(a);
    };
    if (a.by_rows) go(std::true_type{}, std::true_type{});
    else if (a.qt) go(std::false_type{}, std::true_type{});
    else go(std::false_type{}, std::false_type{});
  }
  return launch_status("quant_fp8");
}

Status quant_launch(const TensorDesc* in, int ni, TensorDesc* out, int no, const void* at, void*, size_t,
                    void* stream) {
  if (!quant_sup(in, ni, out, no, at)) return Status::InvalidArgument;
  if (in[0].shape[0] == 0) return Status::Ok;
  if (no_memory(in[0])) return Status::InvalidArgument;
  for (int k = 0; k < no; ++k)
    if (no_memory(out[k])) return Status::InvalidArgument;
  QuantArgs a{};
  a.M = in[0].shape[0];
  a.K = in[0].shape[1];
  a.x = in[0].data;
  matrix_ld(in[0], false, &a.ldx);
  a.q = (uint8_t*)out[0].data;
  matrix_ld(out[0], true, &a.ldq);
  a.s = (float*)out[1].data;
  scale_out(out[1], &a.s_r, &a.s_c);
  a.by_rows = out[1].shape[0] == a.M;
  if (no == 4) {
    a.qt = (uint8_t*)out[2].data;
    matrix_ld(out[2], true, &a.ldqt);
    a.st = (float*)out[3].data;
    scale_out(out[3], &a.st_r, &a.st_c);
    // a matrix of one row has the same S both ways: ST decides
    a.by_rows = a.by_rows && out[3].shape[0] == a.K;
  }
  const AttrBlob& b = blob(at);
  a.pow2 = b.schema_id == AICF_SCHEMA_QFP8 ? field<int32_t>(b, 0) & 1 : 0;
  int ek;
  elem_kind(in[0], &ek);
  const bool e5 = dt(out[0]) == DType::kF8E5M2;
  hipStream_t s = as_stream(stream);
  if (ek == EL_F32) return e5 ? quant_run<EL_F32, 1>(a, s) : quant_run<EL_F32, 0>(a, s);
  if (ek == EL_F16) return e5 ? quant_run<EL_F16, 1>(a, s) : quant_run<EL_F16, 0>(a, s);
  return e5 ? quant_run<EL_BF16, 1>(a, s) : quant_run<EL_BF16, 0>(a, s);
}

size_t no_workspace(const TensorDesc*, int, const void*) { return 0; }

}  // namespace

KernelVariant make_quant_fp8_variant() {
  KernelVariant v;
  v.name = "quant_fp8";
  v.launch = quant_launch;
  v.supported = quant_sup;
  v.query_workspace = no_workspace;
  return v;
}

}  // namespace aicf::hip
