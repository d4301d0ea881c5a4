// Layer norm over the last dimension and its gradients, for gfx950.
//
//   mean = sum x / D;  rstd = 1 / sqrt(sum (x - mean)^2 / D + eps);  n = (x - mean) rstd
//   y = n gamma + beta
//   h = g gamma;  gx = rstd (h - mean(h) - n mean(h n));  ggamma = sum_rows g n;  gbeta = sum_rows g
//
// Bound by memory: a row is read once and held in registers (fp32) by T threads of 8 or
// 16 elements each, so that the deviations are taken from the row's own mean (two passes
// over registers, none over memory).  T is a wave for up to 1024 elements (no barrier), up
// to 1024 threads for 16384; longer rows are walked in memory.  gamma, beta and the
// backward's sums of the columns stay in registers while a workgroup takes its rows in
// turn; the sums leave as one row for each workgroup and a second kernel adds those in
// order, so equal calls give equal bits.
//
// y may be FP8 blocks of 128 columns (block_quant.h), as the product behind it reads
// them: 16 lanes hold a block.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "block_quant.h"

namespace novaq {
namespace {

// Sums of up to two values over T threads (whole waves), in all of them.  `part`: 2 * 16
// float2, used in turn so that one barrier a sum is enough.
template <int T>
__device__ __forceinline__ float2 group_sum(float2 s, float2 (*part)[16], int turn) {
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    s.x += __shfl_xor(s.x, d);
    s.y += __shfl_xor(s.y, d);
  }
  if constexpr (T > 64) {
    const int wave = threadIdx.x >> 6, first = wave / (T / 64) * (T / 64);
    if ((threadIdx.x & 63) == 0) part[turn][wave] = s;
    __syncthreads();
    s = part[turn][first];
#pragma unroll
    for (int w = 1; w < T / 64; ++w) {
      const float2 o = part[turn][first + w];
      s.x += o.x, s.y += o.y;
    }
  }
  return s;
}

// 8 values stored at column c < D of a row of D.
template <int OT, bool VEC>
__device__ __forceinline__ void out8(void* y, int64_t row, int64_t c, int64_t D,
                                     const float (&v)[8]) {
  if constexpr (VEC) {
    bq_store8<OT, true>(y, row * D + c, 8, v);
  } else if (c + 8 <= D) {
    Raw8<OT> r;
#pragma unroll
    for (int k = 0; k < (int)(sizeof(r) / 4); ++k) {
      if constexpr (OT == F32) r.w[k] = f2u(v[k]);
      else if constexpr (OT == BF16) r.w[k] = pack_bf16x2(f2u(v[2 * k]), f2u(v[2 * k + 1]));
      else r.w[k] = bq_half_bits(v[2 * k]) | bq_half_bits(v[2 * k + 1]) << 16;
    }
    __builtin_memcpy(static_cast<uint8_t*>(y) + (row * D + c) * (dtype_bits(OT) / 8), &r, sizeof(r));
  } else {
    bq_store8<OT, false>(y, row * D + c, D - c, v);
  }
}
template <bool VEC>
__device__ __forceinline__ void param8(const float* p, int64_t c, int64_t D, float none,
                                       float (&v)[8]) {
  float w[8];
  row8<F32, VEC>(p, 0, p ? c : D, D, w);
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = p ? w[k] : none;
}

// 8 values stored at column c of a row of y, or (FP8) in the block that 16 lanes hold.
template <int OT, bool VEC>
__device__ __forceinline__ void put8(void* y, uint8_t* e, int64_t row, int64_t c, int64_t D,
                                     float (&v)[8]) {
  if constexpr (OT == E4M3 || OT == E5M2) {
    const int64_t pitch = bq_pitch(D), groups = bq_groups(D);
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) m = max(m, bq_mag(v[k]));
    m = bq_max16(m);
    const bool odd = m >= 0x7F800000u;
    if (odd) {
      m = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) m = max(m, bq_mag_number(v[k], true));
      m = bq_max16(m);
    }
    const int x = bq_exponent<OT>(m);
    const float inv = bq_inverse(x);
    ti_u32x2 w;
    if (odd)
      w = ti_u32x2{bq_encode4<OT, true>(v[0], v[1], v[2], v[3], inv, true),
                   bq_encode4<OT, true>(v[4], v[5], v[6], v[7], inv, true)};
    else
      w = ti_u32x2{bq_encode4<OT, false>(v[0], v[1], v[2], v[3], inv),
                   bq_encode4<OT, false>(v[4], v[5], v[6], v[7], inv)};
    if (c < pitch) *reinterpret_cast<ti_u32x2*>(static_cast<uint8_t*>(y) + row * pitch + c) = w;
    // (lanes past the last block hold nothing: their exponent is 127, as the padding's)
    if ((c & 127) == 0 && c < groups * 128) e[row * groups + (c >> 7)] = (uint8_t)x;
  } else if (c < D) {
    out8<OT, VEC>(y, row, c, D, v);
  }
}

struct NormArgs {
  const void* x;
  const float *gamma, *beta;
  int64_t R, D;
  float eps;
  void* y;
  uint8_t* e;
  float *mean, *rstd;
};

// (FP8: the threads of a row cover its padded exponents too, T * NV * 8 >= groups * 128)
template <int ST, int OT, int T, int NV, bool VEC>
__global__ __launch_bounds__(T < 256 ? 256 : T) void norm_kernel(const NormArgs a) {
  constexpr int G = T < 256 ? 256 / T : 1;
  __shared__ float2 part[2][16];
  const int t = threadIdx.x % T;
  const int64_t D = a.D;
  const float inv = 1.0f / (float)D;
  float gam[NV][8], bet[NV][8];
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    const int64_t c = (int64_t)(n * T + t) * 8;
    param8<VEC>(a.gamma, c, D, 1.0f, gam[n]);
    param8<VEC>(a.beta, c, D, 0.0f, bet[n]);
  }
  for (int64_t r = (int64_t)blockIdx.x * G + threadIdx.x / T; r < a.R;
       r += (int64_t)gridDim.x * G) {
    float v[NV][8];
    float s = 0.0f;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      row8<ST, VEC>(a.x, r, (int64_t)(n * T + t) * 8, D, v[n]);
#pragma unroll
      for (int k = 0; k < 8; ++k) s += v[n][k];
    }
    const float mean = group_sum<T>(float2{s, 0.0f}, part, 0).x * inv;
    float q = 0.0f;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int64_t c = (int64_t)(n * T + t) * 8;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        v[n][k] -= mean;
        if (VEC ? c < D : c + k < D) q += v[n][k] * v[n][k];
      }
    }
    const float var = group_sum<T>(float2{q, 0.0f}, part, 1).x * inv;
    const float rstd = 1.0f / sqrtf(var + a.eps);
    if (t == 0 && a.mean) {
      a.mean[r] = mean;
      a.rstd[r] = rstd;
    }
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int64_t c = (int64_t)(n * T + t) * 8;
      float y[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        y[k] = v[n][k] * rstd * gam[n][k] + bet[n][k];
        if (OT == E4M3 || OT == E5M2)  // (what lies past the row has no part in a block)
          y[k] = c + k < D ? y[k] : 0.0f;
      }
      put8<OT, VEC>(a.y, a.e, r, c, D, y);
    }
  }
}

// Rows that no workgroup holds: walked three times (the second and third from cache).
template <int ST, int OT, bool VEC>
__global__ __launch_bounds__(1024) void norm_long_kernel(const NormArgs a) {
  __shared__ float2 part[2][16];
  const int64_t D = a.D, end = OT == E4M3 || OT == E5M2 ? bq_groups(D) * 128 : D;
  for (int64_t r = blockIdx.x; r < a.R; r += gridDim.x) {
    float s = 0.0f, q = 0.0f, v[8];
    for (int64_t c = threadIdx.x * 8; c < D; c += 8192) {
      row8<ST, VEC>(a.x, r, c, D, v);
#pragma unroll
      for (int k = 0; k < 8; ++k) s += v[k];
    }
    const float mean = group_sum<1024>(float2{s, 0.0f}, part, 0).x / (float)D;
    for (int64_t c = threadIdx.x * 8; c < D; c += 8192) {
      row8<ST, VEC>(a.x, r, c, D, v);
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (c + k < D) q += (v[k] - mean) * (v[k] - mean);
    }
    const float var = group_sum<1024>(float2{q, 0.0f}, part, 1).x / (float)D;
    const float rstd = 1.0f / sqrtf(var + a.eps);
    if (threadIdx.x == 0 && a.mean) {
      a.mean[r] = mean;
      a.rstd[r] = rstd;
    }
    // (whole rounds of 128 columns: the 16 lanes of a block come here together)
    for (int64_t c = threadIdx.x * 8; c < end; c += 8192) {
      float g[8], b[8];
      row8<ST, VEC>(a.x, r, c, D, v);
      param8<VEC>(a.gamma, c, D, 1.0f, g);
      param8<VEC>(a.beta, c, D, 0.0f, b);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        v[k] = (v[k] - mean) * rstd * g[k] + b[k];
        v[k] = c + k < D ? v[k] : 0.0f;
      }
      put8<OT, VEC>(a.y, a.e, r, c, D, v);
    }
    __syncthreads();
  }
}

struct NormGradArgs {
  const void *g, *x;
  const float *gamma, *mean, *rstd;
  int64_t R, D;
  void* gx;
  float* sums;  // (workgroups, 2, D): of g n, and of g
};

// 1024 / T groups of threads a workgroup, each with a row at a time; their sums meet in
// LDS at the end.  GT: the gradient's type; gx is in x's.
template <int ST, int GT, int T, bool VEC>
__global__ __launch_bounds__(1024) void norm_grad_kernel(const NormGradArgs a) {
  constexpr int G = 1024 / T;
  __shared__ float2 part[2][16];
  __shared__ float join[G > 1 ? 8 * 1024 : 1];
  const int t = threadIdx.x % T, grp = threadIdx.x / T;
  const int64_t D = a.D, stride = (int64_t)gridDim.x * G, c = t * 8;
  const float inv = 1.0f / (float)D;
  float gam[8], sw[8], sb[8];
  param8<VEC>(a.gamma, c, D, 1.0f, gam);
#pragma unroll
  for (int k = 0; k < 8; ++k) sw[k] = sb[k] = 0.0f;
  // A row's loads are on their way while the one before it is summed.
  Raw8<ST> rx;
  Raw8<GT> rg;
  float rm, rr;
  auto fetch = [&](int64_t r) {
    const bool in = r < a.R;
    rx = raw8<ST, VEC>(a.x, r, in ? c : D, D);
    rg = raw8<GT, VEC>(a.g, r, in ? c : D, D);
    rm = in ? a.mean[r] : 0.0f;
    rr = in ? a.rstd[r] : 0.0f;
  };
  fetch((int64_t)blockIdx.x * G + grp);
  // (every group goes through the same number of rounds: they share the barriers)
  int turn = 0;
  for (int64_t r0 = (int64_t)blockIdx.x * G; r0 < a.R; r0 += stride, turn ^= 1) {
    const int64_t r = r0 + grp;
    const bool in = r < a.R;
    float g[8], x[8];
    values8<ST>(rx, x);
    values8<GT>(rg, g);
    const float mean = rm, rstd = rr;
    fetch(r + stride);
    float2 s{0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      x[k] = (x[k] - mean) * rstd;
      sw[k] += g[k] * x[k];
      sb[k] += g[k];
      g[k] *= gam[k];
      s.x += g[k];
      s.y += g[k] * x[k];
    }
    s = group_sum<T>(s, part, turn);
    s.x *= inv, s.y *= inv;
    if (in && a.gx && c < D) {
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] = rstd * (g[k] - s.x - x[k] * s.y);
      out8<ST, VEC>(a.gx, r, c, D, x);
    }
  }
  float* out = a.sums + (int64_t)blockIdx.x * 2 * D;
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    if constexpr (G > 1) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 8; ++i) join[i * 1024 + threadIdx.x] = p ? sb[i] : sw[i];
      __syncthreads();
      // (column 8 (u % T) + u / T of the row: the groups' sums in order)
      for (int u = threadIdx.x; u < 8 * T; u += 1024) {
        const int i = u / T, k = u % T;
        float s = join[i * 1024 + k];
#pragma unroll
        for (int o = 1; o < G; ++o) s += join[i * 1024 + o * T + k];
        if (k * 8 + i < D) out[p * D + k * 8 + i] = s;
      }
    } else if (c < D) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = p ? sb[i] : sw[i];
      store8<F32, VEC>(out + p * D, c, D - c, v);
    }
  }
}

// The gradient of x for rows that no workgroup holds.
template <int ST, int GT, bool VEC>
__global__ __launch_bounds__(1024) void norm_grad_long_kernel(const NormGradArgs a) {
  __shared__ float2 part[2][16];
  const int64_t D = a.D;
  int turn = 0;
  for (int64_t r = blockIdx.x; r < a.R; r += gridDim.x, turn ^= 1) {
    const float mean = a.mean[r], rstd = a.rstd[r];
    float2 s{0.0f, 0.0f};
    float x[8], g[8], w[8];
    for (int64_t c = threadIdx.x * 8; c < D; c += 8192) {
      row8<ST, VEC>(a.x, r, c, D, x);
      row8<GT, VEC>(a.g, r, c, D, g);
      param8<VEC>(a.gamma, c, D, 1.0f, w);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (c + k >= D) continue;
        const float h = g[k] * w[k];
        s.x += h;
        s.y += h * ((x[k] - mean) * rstd);
      }
    }
    s = group_sum<1024>(s, part, turn);
    s.x /= (float)D, s.y /= (float)D;
    for (int64_t c = threadIdx.x * 8; c < D; c += 8192) {
      row8<ST, VEC>(a.x, r, c, D, x);
      row8<GT, VEC>(a.g, r, c, D, g);
      param8<VEC>(a.gamma, c, D, 1.0f, w);
#pragma unroll
      for (int k = 0; k < 8; ++k)
        x[k] = rstd * (g[k] * w[k] - s.x - (x[k] - mean) * rstd * s.y);
      out8<ST, VEC>(a.gx, r, c, D, x);
    }
  }
}

// The columns' sums of such rows: a workgroup (y) has the rows y, y + gridDim.y ..
template <int ST, int GT>
__global__ __launch_bounds__(256) void norm_grad_columns_kernel(const NormGradArgs a) {
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x, D = a.D;
  if (c >= D) return;
  auto at = [&](const void* p, int type, int64_t i) {
    if (type == F32) return static_cast<const float*>(p)[i];
    const uint32_t w = static_cast<const uint16_t*>(p)[i];
    return u2f(type == F16 ? dec_f16(w) : dec_bf16(w));
  };
  float w = 0.0f, b = 0.0f;
  for (int64_t r = blockIdx.y; r < a.R; r += gridDim.y) {
    const float g = at(a.g, GT, r * D + c);
    w += g * ((at(a.x, ST, r * D + c) - a.mean[r]) * a.rstd[r]);
    b += g;
  }
  a.sums[(int64_t)blockIdx.y * 2 * D + c] = w;
  a.sums[(int64_t)blockIdx.y * 2 * D + D + c] = b;
}

// The sums (n, 2, D) added over n.
__global__ __launch_bounds__(1024) void norm_join_kernel(const float* __restrict__ sums, int64_t n,
                                                         int64_t D, float* __restrict__ gw,
                                                         float* __restrict__ gb) {
  __shared__ float part[16][64];
  const int64_t c = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63);
  const float s = bq_join_rows(sums, n, 2 * D, c, part);
  if (threadIdx.x >= 64 || c >= 2 * D) return;
  if (c < D) {
    if (gw) gw[c] = s;
  } else if (gb) {
    gb[c - D] = s;
  }
}

// Threads a row: the fewest that hold it with 16 elements each (8 up to 512 and 2048).
template <class F>
int by_width(int64_t D, F&& f) {
#define NOVAQ_SHAPE(T, NV) f(std::integral_constant<int, T>{}, std::integral_constant<int, NV>{})
  if (D <= 512) return NOVAQ_SHAPE(64, 1);
  if (D <= 1024) return NOVAQ_SHAPE(64, 2);
  if (D <= 2048) return NOVAQ_SHAPE(256, 1);
  if (D <= 4096) return NOVAQ_SHAPE(256, 2);
  if (D <= 8192) return NOVAQ_SHAPE(512, 2);
  return NOVAQ_SHAPE(1024, 2);
#undef NOVAQ_SHAPE
}
constexpr int64_t HELD = 16384;  // the longest row that threads hold

// The backward holds 40 values for each 8 columns: 8 a thread, so that 1024 threads have
// the registers.
template <class F>
int by_width_grad(int64_t D, F&& f) {
  if (D <= 512) return f(std::integral_constant<int, 64>{});
  if (D <= 1024) return f(std::integral_constant<int, 128>{});
  if (D <= 2048) return f(std::integral_constant<int, 256>{});
  if (D <= 4096) return f(std::integral_constant<int, 512>{});
  return f(std::integral_constant<int, 1024>{});
}
constexpr int64_t GRAD_HELD = 8192;

template <class F>
int norm_types(int st, int gt, F&& f) {
#define NOVAQ_TYPES(S, G) f(std::integral_constant<int, S>{}, std::integral_constant<int, G>{})
  if (st == F32) return NOVAQ_TYPES(F32, F32);
  if (st == F16) return gt == F16 ? NOVAQ_TYPES(F16, F16) : NOVAQ_TYPES(F16, F32);
  return gt == BF16 ? NOVAQ_TYPES(BF16, BF16) : NOVAQ_TYPES(BF16, F32);
#undef NOVAQ_TYPES
}

// Workgroups of the backward, and with them the rows of sums: one a CU (16384 x 4096 bf16, both
// launches: 91 us so, 93 with two).
int64_t grad_groups(int64_t R, int64_t D) {
  if (D > GRAD_HELD) return std::min<int64_t>(R, 64);
  int64_t rows = 1;
  by_width_grad(D, [&](auto t_) {
    rows = 1024 / decltype(t_)::value;
    return 0;
  });
  return std::min<int64_t>((R + rows - 1) / rows, 256);
}

template <int ST, int OT>
int forward(const NormArgs& a, hipStream_t st) {
  const bool vec = a.D % 8 == 0;
  if (a.D > HELD) {
    const dim3 grid((unsigned)std::min<int64_t>(a.R, 1 << 16));
    if (vec) hipLaunchKernelGGL((norm_long_kernel<ST, OT, true>), grid, dim3(1024), 0, st, a);
    else hipLaunchKernelGGL((norm_long_kernel<ST, OT, false>), grid, dim3(1024), 0, st, a);
    return check_launch();
  }
  return by_width(a.D, [&](auto t_, auto nv_) {
    constexpr int T = decltype(t_)::value, NV = decltype(nv_)::value;
    constexpr int WG = T < 256 ? 256 : T, G = WG / T;
    // Two rows for each wave or group of them, in at most 8192 workgroups (16384 x 4096 bf16
    // 41.6 us, in 2048 45.9, in 16384 44.5; 4096 x 8192 in 2048 23.6, a row each 26.0).
    const int64_t all = (a.R + G - 1) / G;
    const dim3 grid((unsigned)std::min(all, std::clamp<int64_t>(all / 2, 2048, 8192)));
    if (vec) hipLaunchKernelGGL((norm_kernel<ST, OT, T, NV, true>), grid, dim3(WG), 0, st, a);
    else hipLaunchKernelGGL((norm_kernel<ST, OT, T, NV, false>), grid, dim3(WG), 0, st, a);
    return check_launch();
  });
}

}  // namespace

int layer_norm_launch(const void* x, int x_dtype, int64_t R, int64_t D, const float* gamma,
                      const float* beta, float eps, void* y, int y_dtype, void* exponents,
                      float* mean, float* rstd, hipStream_t st) {
  const NormArgs a{x, gamma, beta, R, D, eps, y, static_cast<uint8_t*>(exponents), mean, rstd};
  auto out = [&](auto st_) {
    constexpr int ST = decltype(st_)::value;
    switch (y_dtype) {
      case F32: return forward<ST, F32>(a, st);
      case F16: return forward<ST, F16>(a, st);
      case BF16: return forward<ST, BF16>(a, st);
      case E4M3: return forward<ST, E4M3>(a, st);
      default: return forward<ST, E5M2>(a, st);
    }
  };
  switch (x_dtype) {
    case F32: return out(std::integral_constant<int, F32>{});
    case F16: return out(std::integral_constant<int, F16>{});
    default: return out(std::integral_constant<int, BF16>{});
  }
}

size_t layer_norm_backward_workspace(int64_t R, int64_t D) {
  return (size_t)grad_groups(R, D) * 2 * (size_t)D * sizeof(float);
}

int layer_norm_backward_launch(const void* g, int g_dtype, const void* x, int x_dtype, int64_t R,
                               int64_t D, const float* gamma, const float* mean,
                               const float* rstd, void* gx, float* gw, float* gb, void* workspace,
                               hipStream_t st) {
  const NormGradArgs a{g, x, gamma, mean, rstd, R, D, gx, static_cast<float*>(workspace)};
  const int64_t groups = grad_groups(R, D);
  const bool vec = D % 8 == 0;
  const int rc = norm_types(x_dtype, g_dtype, [&](auto st_, auto gt_) {
    constexpr int ST = decltype(st_)::value, GT = decltype(gt_)::value;
    if (D > GRAD_HELD) {
      const dim3 grid((unsigned)std::min<int64_t>(R, 1 << 16));
      if (gx) {
        if (vec)
          hipLaunchKernelGGL((norm_grad_long_kernel<ST, GT, true>), grid, dim3(1024), 0, st, a);
        else
          hipLaunchKernelGGL((norm_grad_long_kernel<ST, GT, false>), grid, dim3(1024), 0, st, a);
        const int rl = check_launch();
        if (rl != NOVAQ_OK) return rl;
      }
      hipLaunchKernelGGL((norm_grad_columns_kernel<ST, GT>),
                         dim3((unsigned)((D + 255) / 256), (unsigned)groups), dim3(256), 0, st, a);
      return check_launch();
    }
    return by_width_grad(D, [&](auto t_) {
      constexpr int T = decltype(t_)::value;
      const dim3 grid((unsigned)groups);
      if (vec)
        hipLaunchKernelGGL((norm_grad_kernel<ST, GT, T, true>), grid, dim3(1024), 0, st,
                           a);
      else
        hipLaunchKernelGGL((norm_grad_kernel<ST, GT, T, false>), grid, dim3(1024), 0, st,
                           a);
      return check_launch();
    });
  });
  if (rc != NOVAQ_OK || (!gw && !gb)) return rc;
  hipLaunchKernelGGL(norm_join_kernel, dim3((unsigned)((2 * D + 63) / 64)), dim3(1024), 0, st,
                     static_cast<const float*>(workspace), groups, D, gw, gb);
  return check_launch();
}

}  // namespace novaq
