// FP8 blocks: a power-of-two scale, kept as its exponent e (the scale is 2^(e - 127)), for
// 128 columns of a row or for 128 x 128 elements.  The exponent is the smallest with the
// block's largest finite magnitude within the format's, from integer operations on that
// magnitude's bits: x / scale is then exact in fp32, so a code has one rounding, and
// blocks of equal magnitudes have equal exponents in every implementation.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "novaq_convert.h"
#include "novaq_internal.h"
#include "token_io.h"

namespace novaq {
namespace {

constexpr int BQ = 128;  // elements of a block along a row (and down a column)

// Exponents a row of n elements has: one for 128, in whole fours (the products read them
// as dwords); those past the last block are 127.
__host__ __device__ inline int64_t bq_groups(int64_t n) { return ((n + 127) / 128 + 3) / 4 * 4; }
__host__ __device__ inline int64_t bq_pitch(int64_t n) { return (n + 127) / 128 * 128; }

// fp16 by the hardware's conversions, one instruction each where those of the casts, which
// keep a NaN's payload, are 6 and 14 (a norm of 16384 x 4096 fp16 66 us with them, so 42; a
// product of 8192 x 16384 x 1024 219 and 157).
__device__ __forceinline__ float bq_half(uint32_t h) {
  return (float)__builtin_bit_cast(_Float16, (uint16_t)h);
}
__device__ __forceinline__ uint32_t bq_half_bits(float v) {
  return __builtin_bit_cast(uint16_t, (_Float16)v);
}
// A 16-bit value as stored, in fp32.
template <int ST>
__device__ __forceinline__ float bq_value16(uint32_t c) {
  if constexpr (ST == F16) return bq_half(c);
  else return u2f(decode<ST>(c));
}
// 8 values stored as token_io.h's store8 does.
template <int OT, bool VEC>
__device__ __forceinline__ void bq_store8(void* out, int64_t e, int64_t left, const float (&v)[8]) {
  if constexpr (OT == F16) {
    uint16_t* p = static_cast<uint16_t*>(out) + e;
    if constexpr (VEC) {
      ti_u32x4 a;
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = bq_half_bits(v[2 * i]) | bq_half_bits(v[2 * i + 1]) << 16;
      *reinterpret_cast<ti_u32x4*>(p) = a;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < left) p[i] = (uint16_t)bq_half_bits(v[i]);
    }
  } else {
    store8<OT, VEC>(out, e, left, v);
  }
}

// 8 columns from c on of a row of D as stored, zeros past it.  VEC: the rows start on 16
// bytes; otherwise whole runs are still one access (of any alignment: 16384 rows of 500
// bf16 30 us a value at a time).
template <int ST>
struct Raw8 {
  uint32_t w[ST == F32 ? 8 : 4];
};
template <int ST, bool VEC>
__device__ __forceinline__ Raw8<ST> raw8(const void* x, int64_t row, int64_t c, int64_t D) {
  constexpr int SIZE = dtype_bits(ST) / 8;
  Raw8<ST> r;
#pragma unroll
  for (int k = 0; k < (int)(sizeof(r) / 4); ++k) r.w[k] = 0;
  const uint8_t* p = static_cast<const uint8_t*>(x) + (row * D + c) * SIZE;
  if (c + 8 <= D) {
    if constexpr (VEC) {
#pragma unroll
      for (int k = 0; k < (int)(sizeof(r) / 16); ++k) {
        const ti_u32x4 a = reinterpret_cast<const ti_u32x4*>(p)[k];
#pragma unroll
        for (int i = 0; i < 4; ++i) r.w[4 * k + i] = a[i];
      }
    } else {
      __builtin_memcpy(&r, p, sizeof(r));
    }
  } else if (!VEC && c < D) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (c + k < D) {
        if constexpr (ST == F32) r.w[k] = reinterpret_cast<const uint32_t*>(p)[k];
        else r.w[k / 2] |= (uint32_t) reinterpret_cast<const uint16_t*>(p)[k] << (16 * (k & 1));
      }
    }
  }
  return r;
}
template <int ST>
__device__ __forceinline__ void values8(const Raw8<ST>& r, float (&v)[8]) {
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    if constexpr (ST == F32) v[k] = u2f(r.w[k]);
    else v[k] = bq_value16<ST>(r.w[k / 2] >> (16 * (k & 1)) & 0xFFFFu);
  }
}
template <int ST, bool VEC>
__device__ __forceinline__ void row8(const void* x, int64_t row, int64_t c, int64_t D,
                                     float (&v)[8]) {
  values8<ST>(raw8<ST, VEC>(x, row, c, D), v);
}

// Magnitude bits a (not NaN) -> exponent.  The largest codes are 1.75 * 2^8 and 1.75 *
// 2^15.  Nothing and infinity give 127 (a scale of 1), as per-tensor scales do.
template <int DT>
__device__ __forceinline__ int bq_exponent(uint32_t a) {
  const int e = (int)(a >> 23) - (DT == E4M3 ? 8 : 15) + ((a & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return a == 0 || a >= 0x7F800000u ? 127 : max(e, 1);
}

// 1 / scale (exponents are 1 .. 247: a normal number).
__device__ __forceinline__ float bq_inverse(int e) { return u2f((uint32_t)(254 - e) << 23); }
__device__ __forceinline__ float bq_scale(int e) { return u2f((uint32_t)e << 23); }

// max |v| as bits, a NaN counted as more than an infinity.
__device__ __forceinline__ uint32_t bq_mag(float v) { return f2u(v) & 0x7FFFFFFFu; }
// The same with NaNs (and infinities, where they become NaNs) passed over: blocks that hold
// one are looked at again.
__device__ __forceinline__ uint32_t bq_mag_number(float v, bool inf_nan = false) {
  const uint32_t a = bq_mag(v);
  return a > (inf_nan ? 0x7F7FFFFFu : 0x7F800000u) ? 0u : a;
}

// max over the 16 lanes of a row of lanes, in all of them.
__device__ __forceinline__ uint32_t bq_max16(uint32_t a) {
#define NOVAQ_ROR(N) \
  a = max(a, (uint32_t)__builtin_amdgcn_mov_dpp((int)a, 0x120 + (N), 0xF, 0xF, true))
  NOVAQ_ROR(1);
  NOVAQ_ROR(2);
  NOVAQ_ROR(4);
  NOVAQ_ROR(8);
#undef NOVAQ_ROR
  return a;
}

// 4 codes of v * inv.  ODD: the block may hold an infinity or a NaN: the casts' rule
// saturates the first, and the second keeps its sign and has all other bits of its code
// set, which the hardware's conversion does not do; in all others nothing exceeds the
// largest code.  inf_nan: an infinity becomes such a NaN too, what the layers' own operands
// are made with: a gradient that has overflowed must not come out of a product finite.
template <int DT, bool ODD>
__device__ __forceinline__ uint32_t bq_encode4(float a, float b, float c, float d, float inv,
                                               bool inf_nan = false) {
  a *= inv, b *= inv, c *= inv, d *= inv;
  uint32_t nan = 0;
  if constexpr (ODD) {
    auto bound = [&](float v, int at) {
      const float t = __builtin_amdgcn_fmed3f(v, -fmt_max(DT), fmt_max(DT));
      const bool number = inf_nan ? fabsf(v) <= fmt_max(DT) : v == v;
      nan |= number ? 0u : (0x7Fu | (f2u(v) >> 24 & 0x80u)) << at;
      return number ? t : 0.0f;
    };
    a = bound(a, 0), b = bound(b, 8), c = bound(c, 16), d = bound(d, 24);
  }
  int w = 0;
  if constexpr (DT == E4M3) {
    w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, w, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
  } else {
    w = __builtin_amdgcn_cvt_pk_bf8_f32(a, b, w, false);
    w = __builtin_amdgcn_cvt_pk_bf8_f32(c, d, w, true);
  }
  return (uint32_t)w | nan;
}

// Column c of sums (n, C) added over n by a workgroup of 16 waves, 64 columns: each wave has
// every 16th row, and wave 0 the sum (with 4 waves and a row in flight each 64 x 4096 took 6.5
// us, so 3.9).
__device__ __forceinline__ float bq_join_rows(const float* __restrict__ sums, int64_t n, int64_t C,
                                              int64_t c, float (*part)[64]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float s = 0.0f;
  if (c < C) {
#pragma unroll 4
    for (int64_t i = wave; i < n; i += 16) s += sums[i * C + c];
  }
  part[wave][lane] = s;
  __syncthreads();
  if (wave != 0) return 0.0f;
#pragma unroll
  for (int w = 1; w < 16; ++w) s += part[w][lane];
  return s;
}

// Where the blocks of one R x C matrix go; codes or codes_t may be null.
struct BlockOut {
  uint8_t *codes, *e;      // (R, pitch(C)), exponents (R or R / 128 up, groups(C))
  uint8_t *codes_t, *et;   // (C, pitch(R)), exponents (C or C / 128 up, groups(R))
};

constexpr int BQ_THREADS = 512, BQ_WAVES = BQ_THREADS / 64, BQ_R = BQ * 16 / BQ_THREADS;
struct BlockTileLds {
  uint8_t t[BQ * BQ];  // the transposed codes
  uint32_t top[BQ_WAVES][BQ];
  float sum[BQ_WAVES][BQ];
};

// The place of the four codes of column c, rows 4 g .. + 3 in LDS: rows of 128 bytes whose
// 16-byte chunks are exchanged, so that a wave's stores (16 columns 8 apart, 4 fours) meet
// in a bank twice and not 8 times.
__device__ __forceinline__ int bq_slot(int c, int chunk) {
  return c * BQ + ((chunk ^ (c >> 3 & 7)) << 4);
}

// One 128 x 128 tile (rt, ct) of a matrix by 512 threads: thread t holds rows 4 (t / 16) ..
// + 3, columns 8 (t % 16) .. + 7 in v, zeros past the matrix (with 256 threads of 8 rows
// the registers leave two waves a SIMD).  TILE: one exponent for the tile, else one for
// each row (codes) and one for each column (codes_t).  ODD: the tile holds an infinity or
// a NaN; inf_nan as in bq_encode4.  colsum (this tile row's partial sums, or null).  All
// threads come here.
template <int DT, bool TILE, bool ODD>
__device__ __forceinline__ void bq_tile_as(const float (&v)[BQ_R][8], int64_t R, int64_t C,
                                           int64_t rt, int64_t ct, const BlockOut& o,
                                           float* colsum, BlockTileLds& lds, bool inf_nan) {
  const int tid = threadIdx.x, rg = tid >> 4, cg = tid & 15, wave = tid >> 6;
  const int64_t r0 = rt * BQ + rg * BQ_R, c0 = ct * BQ + cg * 8;
  const int64_t groups = bq_groups(C), groups_t = bq_groups(R);
  const int64_t last = (C + 127) / 128 - 1, last_t = (R + 127) / 128 - 1;
  auto mag = [&](float f) { return ODD ? bq_mag_number(f, inf_nan) : bq_mag(f); };
  int te = 0;
  if constexpr (TILE) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < BQ_R; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) m = max(m, mag(v[i][j]));
#pragma unroll
    for (int d = 32; d; d >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, d));
    if ((tid & 63) == 0) lds.top[0][wave] = m;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < BQ_WAVES; ++k) m = max(m, lds.top[0][k]);
    te = bq_exponent<DT>(m);
  }
  if (o.codes) {
    uint8_t* to = o.codes + r0 * bq_pitch(C) + c0;
#pragma unroll
    for (int i = 0; i < BQ_R; ++i) {
      int e = te;
      if constexpr (!TILE) {
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max(m, mag(v[i][j]));
        e = bq_exponent<DT>(bq_max16(m));
      }
      const float inv = bq_inverse(e);
      const ti_u32x2 w{bq_encode4<DT, ODD>(v[i][0], v[i][1], v[i][2], v[i][3], inv, inf_nan),
                       bq_encode4<DT, ODD>(v[i][4], v[i][5], v[i][6], v[i][7], inv, inf_nan)};
      if (r0 + i < R) {
        *reinterpret_cast<ti_u32x2*>(to + i * bq_pitch(C)) = w;
        if (cg == 0 && (!TILE || (rg == 0 && i == 0))) {
          uint8_t* at = o.e + (TILE ? rt : r0 + i) * groups + ct;
          *at = (uint8_t)e;
          if (ct == last)
            for (int64_t k = ct + 1; k < groups; ++k) *++at = 127;
        }
      }
    }
  }
  if (o.codes_t) {
    uint32_t col[8];
    if constexpr (!TILE) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        col[j] = 0;
#pragma unroll
        for (int i = 0; i < BQ_R; ++i) col[j] = max(col[j], mag(v[i][j]));
        col[j] = max(col[j], (uint32_t)__shfl_xor((int)col[j], 16));
        col[j] = max(col[j], (uint32_t)__shfl_xor((int)col[j], 32));
        if ((tid & 48) == 0) lds.top[wave][cg * 8 + j] = col[j];
      }
      __syncthreads();
      if (tid < BQ) {
        uint32_t m = lds.top[0][tid];
#pragma unroll
        for (int k = 1; k < BQ_WAVES; ++k) m = max(m, lds.top[k][tid]);
        const int e = bq_exponent<DT>(m);
        lds.top[0][tid] = (uint32_t)e;
        if (ct * BQ + tid < C) {
          uint8_t* at = o.et + (ct * BQ + tid) * groups_t + rt;
          *at = (uint8_t)e;
          if (rt == last_t)
            for (int64_t k = rt + 1; k < groups_t; ++k) *++at = 127;
        }
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 8; ++j) col[j] = lds.top[0][cg * 8 + j];
    } else if (tid == 0) {
      uint8_t* at = o.et + ct * groups_t + rt;
      *at = (uint8_t)te;
      if (rt == last_t)
        for (int64_t k = rt + 1; k < groups_t; ++k) *++at = 127;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float inv = bq_inverse(TILE ? te : (int)col[j]);
      *reinterpret_cast<uint32_t*>(lds.t + bq_slot(cg * 8 + j, rg >> 2) + (rg & 3) * 4) =
          bq_encode4<DT, ODD>(v[0][j], v[1][j], v[2][j], v[3][j], inv, inf_nan);
    }
  }
  if (!TILE && colsum) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float s = (v[0][j] + v[1][j]) + (v[2][j] + v[3][j]);
      s += __shfl_xor(s, 16);
      s += __shfl_xor(s, 32);
      if ((tid & 48) == 0) lds.sum[wave][cg * 8 + j] = s;
    }
  }
  __syncthreads();
  if (o.codes_t) {
    // 8 threads a row of 128 codes, 16 bytes each
#pragma unroll
    for (int k = tid; k < BQ * 8; k += BQ_THREADS) {
      const int c = k >> 3, p = k & 7;
      if (ct * BQ + c < C)
        *reinterpret_cast<ti_u32x4*>(o.codes_t + (ct * BQ + c) * bq_pitch(R) + rt * BQ + p * 16) =
            *reinterpret_cast<const ti_u32x4*>(lds.t + bq_slot(c, p));
    }
  }
  if (!TILE && colsum && tid < BQ && ct * BQ + tid < C)
    colsum[ct * BQ + tid] =
        ((lds.sum[0][tid] + lds.sum[1][tid]) + (lds.sum[2][tid] + lds.sum[3][tid])) +
        ((lds.sum[4][tid] + lds.sum[5][tid]) + (lds.sum[6][tid] + lds.sum[7][tid]));
}

// The same for whatever the tile holds.
template <int DT, bool TILE>
__device__ __forceinline__ void bq_tile(const float (&v)[BQ_R][8], int64_t R, int64_t C, int64_t rt,
                                        int64_t ct, const BlockOut& o, float* colsum,
                                        BlockTileLds& lds, bool inf_nan = false) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < BQ_R; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, bq_mag(v[i][j]));
  if (!__syncthreads_or(m >= 0x7F800000u))
    bq_tile_as<DT, TILE, false>(v, R, C, rt, ct, o, colsum, lds, false);
  else
    bq_tile_as<DT, TILE, true>(v, R, C, rt, ct, o, colsum, lds, inf_nan);
}

// A thread's 4 x 8 part of tile (rt, ct) of x (R, C), zeros past it.
template <int ST, bool VEC>
__device__ __forceinline__ void bq_load(const void* x, int64_t R, int64_t C, int64_t rt,
                                        int64_t ct, float (&v)[BQ_R][8]) {
  const int rg = threadIdx.x >> 4, cg = threadIdx.x & 15;
  const int64_t r0 = rt * BQ + rg * BQ_R, c0 = ct * BQ + cg * 8;
  Raw8<ST> raw[BQ_R];
#pragma unroll
  for (int i = 0; i < BQ_R; ++i) raw[i] = raw8<ST, VEC>(x, r0 + i, r0 + i < R ? c0 : C, C);
#pragma unroll
  for (int i = 0; i < BQ_R; ++i) values8<ST>(raw[i], v[i]);
}

}  // namespace
}  // namespace novaq
