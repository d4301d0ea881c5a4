// Matrices to FP8 blocks and back (block_quant.h has the rule).
//
// Bound by memory: 2 (or 4) bytes an element read, one written for each order of codes.
// A workgroup has a 128 x 128 tile in registers, so one read serves both orders (the
// transposed product's codes and exponents, which are of 128 rows, go through LDS) and
// the columns' sums.  For a few rows, or codes in one order, 16 lanes take a block.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "block_quant.h"

namespace novaq {
namespace {

template <int ST, int DT, bool TILE, bool VEC>
__global__ __launch_bounds__(BQ_THREADS, 6) void block_tile_kernel(const void* __restrict__ x, int64_t R,
                                                         int64_t C, BlockOut o,
                                                         float* __restrict__ sums, bool inf_nan) {
  __shared__ __attribute__((aligned(16))) BlockTileLds lds;
  const int64_t ctiles = (C + 127) / 128;
  const int64_t rt = blockIdx.x / ctiles, ct = blockIdx.x % ctiles;
  if (gridDim.y > 1) {  // each order by workgroups of its own
    if (blockIdx.y == 0) o.codes_t = nullptr, sums = nullptr;
    else o.codes = nullptr;
  }
  float v[BQ_R][8];
  bq_load<ST, VEC>(x, R, C, rt, ct, v);
  bq_tile<DT, TILE>(v, R, C, rt, ct, o, sums ? sums + rt * C : nullptr, lds, inf_nan);
}

// The codes of rows alone: 16 lanes a block of 128 columns, 8 columns a lane.
template <int ST, int DT, bool VEC>
__global__ __launch_bounds__(256) void block_rows_kernel(const void* __restrict__ x, int64_t R,
                                                         int64_t C, uint8_t* __restrict__ codes,
                                                         uint8_t* __restrict__ e, bool inf_nan) {
  const int cg = threadIdx.x & 15;
  const int64_t blocks = (C + 127) / 128, groups = bq_groups(C), pitch = bq_pitch(C);
  const int64_t all = R * blocks, stride = (int64_t)gridDim.x * 16;
  for (int64_t b = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4); b < all; b += stride) {
    const int64_t r = b / blocks, g = b - r * blocks, c = g * 128 + cg * 8;
    float v[8];
    row8<ST, VEC>(x, r, c, C, v);
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, bq_mag(v[j]));
    m = bq_max16(m);
    const bool odd = m >= 0x7F800000u;
    if (odd) {
      m = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) m = max(m, bq_mag_number(v[j], inf_nan));
      m = bq_max16(m);
    }
    const int x_ = bq_exponent<DT>(m);
    const float inv = bq_inverse(x_);
    ti_u32x2 w;
    if (odd)
      w = ti_u32x2{bq_encode4<DT, true>(v[0], v[1], v[2], v[3], inv, inf_nan),
                   bq_encode4<DT, true>(v[4], v[5], v[6], v[7], inv, inf_nan)};
    else
      w = ti_u32x2{bq_encode4<DT, false>(v[0], v[1], v[2], v[3], inv),
                   bq_encode4<DT, false>(v[4], v[5], v[6], v[7], inv)};
    *reinterpret_cast<ti_u32x2*>(codes + r * pitch + c) = w;
    if (cg == 0) {
      e[r * groups + g] = (uint8_t)x_;
      if (g == blocks - 1)
        for (int64_t k = blocks; k < groups; ++k) e[r * groups + k] = 127;
    }
  }
}

// sums (n, C) added over n.
__global__ __launch_bounds__(1024) void block_colsum_kernel(const float* __restrict__ sums,
                                                            int64_t n, int64_t C,
                                                            float* __restrict__ out) {
  __shared__ float part[16][64];
  const int64_t c = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63);
  const float s = bq_join_rows(sums, n, C, c, part);
  if (threadIdx.x < 64 && c < C) out[c] = s;
}

template <int DT, int OT>
__global__ __launch_bounds__(256) void block_decode_kernel(const uint8_t* __restrict__ codes,
                                                           const uint8_t* __restrict__ e,
                                                           int64_t R, int64_t C, int shift,
                                                           void* __restrict__ out, bool vec) {
  const int64_t units = bq_pitch(C) / 8, groups = bq_groups(C), pitch = bq_pitch(C);
  const int64_t all = R * units, stride = (int64_t)gridDim.x * 256;
  for (int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x; u < all; u += stride) {
    const int64_t r = u / units, c = (u - r * units) * 8;
    if (c >= C) continue;
    float v[8];
    load8<DT, true>(codes + r * pitch, c, pitch, v);
    // (a code times 2^(e - 127), rounded once: two factors where the power is not normal)
    const int x = e[(r >> shift) * groups + (c >> 7)];
    const float s = x == 255 ? u2f(0x7FC00000u) : x == 0 ? 0x1p-127f : bq_scale(x);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= s;
    if (vec) bq_store8<OT, true>(out, r * C + c, 8, v);
    else bq_store8<OT, false>(out, r * C + c, min<int64_t>(8, C - c), v);
  }
}

template <class F>
int by_type(int st, F&& f) {
  switch (st) {
    case F32: return f(std::integral_constant<int, F32>{});
    case F16: return f(std::integral_constant<int, F16>{});
    default: return f(std::integral_constant<int, BF16>{});
  }
}
template <class F>
int by_bool(bool b, F&& f) {
  return b ? f(std::true_type{}) : f(std::false_type{});
}
template <class F>
int by_fp8(int dt, F&& f) {
  return dt == E4M3 ? f(std::integral_constant<int, E4M3>{})
                    : f(std::integral_constant<int, E5M2>{});
}

}  // namespace

size_t quantize_blocks_workspace(int64_t R, int64_t C) {
  return (size_t)((R + 127) / 128) * (size_t)C * sizeof(float);
}

int quantize_blocks_launch(const void* x, int x_dtype, int64_t R, int64_t C, int dtype,
                           int block_rows, void* codes, void* e, void* codes_t, void* et,
                           float* colsum, void* workspace, bool inf_nan, hipStream_t st) {
  const bool vec = C % 8 == 0;
  const BlockOut o{static_cast<uint8_t*>(codes), static_cast<uint8_t*>(e),
                   static_cast<uint8_t*>(codes_t), static_cast<uint8_t*>(et)};
  return by_type(x_dtype, [&](auto st_) {
    return by_fp8(dtype, [&](auto dt_) {
      return by_bool(vec, [&](auto vec_) {
        constexpr int ST = decltype(st_)::value, DT = decltype(dt_)::value;
        constexpr bool VEC = decltype(vec_)::value;
        if (block_rows == 1 && !codes_t && !colsum) {
          const int64_t groups = (R * ((C + 127) / 128) + 15) / 16;
          hipLaunchKernelGGL((block_rows_kernel<ST, DT, VEC>),
                             dim3((unsigned)std::min<int64_t>(groups, 1 << 16)), dim3(256), 0, st,
                             x, R, C, o.codes, o.e, inf_nan);
          return check_launch();
        }
        const int64_t rt = (R + 127) / 128, tiles = rt * ((C + 127) / 128);
        float* sums = colsum ? (rt == 1 ? colsum : static_cast<float*>(workspace)) : nullptr;
        // (a few tiles leave CUs idle: 128 x 128 5.5 us so, 6.6 together; 1024 x 2048 8.3 and 9.1;
        // 2048 x 2048 10.3 and 10.2, 2048 x 4096 13.0 and 12.6)
        const unsigned orders = codes && codes_t && tiles <= 128 ? 2 : 1;
        if (block_rows == 1)
          hipLaunchKernelGGL((block_tile_kernel<ST, DT, false, VEC>), dim3((unsigned)tiles, orders),
                             dim3(BQ_THREADS), 0, st, x, R, C, o, sums, inf_nan);
        else
          hipLaunchKernelGGL((block_tile_kernel<ST, DT, true, VEC>), dim3((unsigned)tiles),
                             dim3(BQ_THREADS), 0, st, x, R, C, o, nullptr, inf_nan);
        const int rc = check_launch();
        if (rc != NOVAQ_OK || !sums || rt == 1) return rc;
        hipLaunchKernelGGL(block_colsum_kernel, dim3((unsigned)((C + 63) / 64)), dim3(1024), 0, st,
                           sums, rt, C, colsum);
        return check_launch();
      });
    });
  });
}

int dequantize_blocks_launch(const void* codes, int dtype, const void* e, int64_t R, int64_t C,
                             int block_rows, void* out, int out_dtype, hipStream_t st) {
  const int64_t units = R * (bq_pitch(C) / 8);
  const dim3 grid((unsigned)std::min<int64_t>((units + 255) / 256, 1 << 16));
  return by_fp8(dtype, [&](auto dt_) {
    return by_type(out_dtype, [&](auto ot_) {
      constexpr int DT = decltype(dt_)::value, OT = decltype(ot_)::value;
      hipLaunchKernelGGL((block_decode_kernel<DT, OT>), grid, dim3(256), 0, st,
                         static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(e), R, C,
                         block_rows == 128 ? 7 : 0, out, C % 8 == 0);
      return check_launch();
    });
  });
}

}  // namespace novaq
