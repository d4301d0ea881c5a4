// Clipping of many gradients by their global norm.
//
//   norm = sqrt(sum over all tensors and elements of g^2)
//   out  = g * min(1, max_norm / (norm + eps))
//
// Two passes over memory: the first leaves one fp64 sum of squares a workgroup
// (products and sums in fp64, so neither the largest fp32 gradient nor the
// smallest one leaves the range), the second adds these in a fixed order in
// every workgroup (from L2) and scales.  Both are bound by memory.  The tensors'
// addresses and lengths travel in the kernels' arguments, or, past 120 of them,
// through the workspace, which small kernels fill from theirs: nothing is copied
// from host memory and nothing about a tensor outlives the call.
//
// All tensors are cut into runs (of 2048 to 16384 elements: at most 8 for each of
// 2048 workgroups where there are enough elements), which the workgroups take in
// turn, each looked up by bisection in the tensors' first runs.  A lane loads 4
// vectors before it uses the first.  Loads and stores go past the caches (353M bf16
// gradients: the first pass 167 us with plain loads, 104 = 6.8 TB/s so; 4 and 8 ahead
// alike) and every instruction of a wave covers whole lines (8 gradients a lane to
// two 16-byte stores of fp32: 573 us for the second pass, 390 = 5.4 TB/s with 4).
// Both passes with plain loads and stores, and so: 353M bf16 to fp32 543 and 498 us,
// 133M fp32 314 and 267, 53M bf16 to fp32 74 and 78, 51M f16 66 and 70, 18M bf16 24
// and 24: what the 256 MB cache holds loses 6%, what it does not gains 8 to 15.
// Neither fewer registers nor fp32 products change the times.
//
// The factor is worked out in fp64 too, and float64 gradients are multiplied by it as
// it is; the others by its fp32 rounding (a norm past fp32's range still scales them).
//
// NaN or infinite gradients give a NaN or infinite norm: the factor is then
// NaN or 0, as the formula says (min keeps a NaN).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "novaq_internal.h"
#include "token_io.h"

namespace novaq {
namespace {

constexpr int F64 = NOVAQ_F64;  // (only here: float64 gradients)
constexpr int ROWS = 120;       // tensors in a kernel's arguments (3840 bytes)
constexpr int BLOCKS = 2048;    // workgroups of a pass: eight a CU
constexpr int STEP = 2048;      // elements of a run are a multiple

struct NormRow {
  const void* g;
  void* out;
  int64_t n;
  uint32_t first;  // its first run
  uint8_t gt, ot;
};
static_assert(sizeof(NormRow) == 32, "120 rows fit a kernel's arguments");

struct NormRows {
  NormRow row[ROWS];
};

__global__ __launch_bounds__(128) void norm_rows_kernel(const NormRows l, int count,
                                                        NormRow* __restrict__ table) {
  if ((int)threadIdx.x < count) table[threadIdx.x] = l.row[threadIdx.x];
}

// The tensor that holds run r.
template <class T>
__device__ __forceinline__ int tensor_of(const T& rows, int count, uint32_t r) {
  int lo = 0, hi = count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (rows[mid].first <= r) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ double block_sum(double s, double* part) {
#pragma unroll
  for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  s = part[0] + part[1] + part[2] + part[3];
  __syncthreads();
  return s;
}

// W values (4 or 8) of type GT, one vector load.
template <int GT, int W, bool NT>
__device__ __forceinline__ void load_w(const uint8_t* b, int64_t i, float (&v)[W]) {
  if constexpr (W == 8) {
    load8<GT, true, NT>(b, i, 0, v);
  } else if constexpr (GT == F32) {
    const ti_u32x4 a = vload<NT>(reinterpret_cast<const ti_u32x4*>(b + i * 4));
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = u2f(a[k]);
  } else {
    const ti_u32x2 a = vload<NT>(reinterpret_cast<const ti_u32x2*>(b + i * 2));
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const uint32_t w = a[k];
      v[2 * k] = u2f(decode<GT>(w & 0xFFFFu));
      v[2 * k + 1] = u2f(decode<GT>(w >> 16));
    }
  }
}

template <int OT, int W, bool NT>
__device__ __forceinline__ void store_w(void* out, int64_t i, const float (&v)[W]) {
  if constexpr (W == 8) {
    store8<OT, true, NT>(out, i, 8, v);
  } else if constexpr (OT == F32) {
    vstore<NT>(reinterpret_cast<ti_u32x4*>(reinterpret_cast<float*>(out) + i),
                 ti_u32x4{f2u(v[0]), f2u(v[1]), f2u(v[2]), f2u(v[3])});
  } else {
    ti_u32x2 a;
#pragma unroll
    for (int k = 0; k < 2; ++k)
      a[k] = encode<OT>(f2u(v[2 * k])) | (encode<OT>(f2u(v[2 * k + 1])) << 16);
    vstore<NT>(reinterpret_cast<ti_u32x2*>(reinterpret_cast<uint16_t*>(out) + i), a);
  }
}

// Elements e0 .. e1 - 1 (e0 a multiple of 2048): fw(i, v) gets W values from
// element i on, f1(i, v) one.  W values are one vector of at most 16 bytes, so
// that every load of a wave covers whole lines.  Without `vec` f1 gets them all.
template <int GT, int W, bool NT, class FW, class F1>
__device__ __forceinline__ void each_of_run(const void* p, int64_t e0, int64_t e1, bool vec,
                                            FW&& fw, F1&& f1) {
  const uint8_t* b = static_cast<const uint8_t*>(p);
  int64_t i = e0;
  if constexpr (GT != F64) {
    if (vec && (reinterpret_cast<uintptr_t>(b) & 15) == 0) {
      constexpr int S = 256 * W, A = 4;  // elements of a step; vectors ahead
      for (; i + A * S <= e1; i += A * S) {
        float v[A][W];
#pragma unroll
        for (int k = 0; k < A; ++k) load_w<GT, W, NT>(b, i + k * S + threadIdx.x * W, v[k]);
#pragma unroll
        for (int k = 0; k < A; ++k) fw(i + k * S + threadIdx.x * W, v[k]);
      }
      const int64_t whole = i + (e1 - i) / W * W;
      for (int64_t k = i + threadIdx.x * W; k < whole; k += S) {
        float v[W];
        load_w<GT, W, NT>(b, k, v);
        fw(k, v);
      }
      i = whole;
    }
  }
  for (int64_t k = i + threadIdx.x; k < e1; k += 256) {
    if constexpr (GT == F64) f1(k, reinterpret_cast<const double*>(b)[k]);
    else if constexpr (GT == F32) f1(k, reinterpret_cast<const float*>(b)[k]);
    else f1(k, u2f(decode<GT>(reinterpret_cast<const uint16_t*>(b)[k])));
  }
}

template <class T>
__device__ __forceinline__ double sum_runs(const T& rows, int count, uint32_t runs, int run) {
  double s = 0.0;
  for (uint32_t r = blockIdx.x; r < runs; r += gridDim.x) {
    const int t = tensor_of(rows, count, r);
    const int64_t e0 = (int64_t)(r - rows[t].first) * run, e1 = min(rows[t].n, e0 + run);
    auto add_w = [&](int64_t, const auto& v) {
#pragma unroll
      for (int k = 0; k < (int)(sizeof(v) / 4); ++k) s = fma((double)v[k], (double)v[k], s);
    };
    auto add_1 = [&](int64_t, auto v) { s = fma((double)v, (double)v, s); };
    const void* g = rows[t].g;
    switch (rows[t].gt) {
      case F32: each_of_run<F32, 4, true>(g, e0, e1, true, add_w, add_1); break;
      case F16: each_of_run<F16, 8, true>(g, e0, e1, true, add_w, add_1); break;
      case BF16: each_of_run<BF16, 8, true>(g, e0, e1, true, add_w, add_1); break;
      default: each_of_run<F64, 8, true>(g, e0, e1, true, add_w, add_1); break;
    }
  }
  return s;
}

template <bool TABLE>
__global__ __launch_bounds__(256) void norm_sum_kernel(const NormRows l,
                                                       const NormRow* __restrict__ table,
                                                       int count, uint32_t runs, int run,
                                                       double* __restrict__ slots) {
  __shared__ double part[4];
  double s;
  if constexpr (TABLE) s = sum_runs(table, count, runs, run);
  else s = sum_runs(l.row, count, runs, run);
  s = block_sum(s, part);
  if (threadIdx.x == 0) slots[blockIdx.x] = s;
}

template <int OT>
__device__ __forceinline__ void put(void* out, int64_t i, float v) {
  if constexpr (OT == F32) reinterpret_cast<float*>(out)[i] = v;
  else if constexpr (OT == F64) reinterpret_cast<double*>(out)[i] = (double)v;
  else reinterpret_cast<uint16_t*>(out)[i] = (uint16_t)encode<OT>(f2u(v));
}
template <int GT, int OT>
__device__ __forceinline__ void scale_run(const void* g, void* out, int64_t e0, int64_t e1,
                                          double coef64) {
  constexpr int W = GT == F32 || OT == F32 ? 4 : 8;
  const float coef = (float)coef64;
  each_of_run<GT, W, true>(
      g, e0, e1, OT != F64 && (reinterpret_cast<uintptr_t>(out) & 15) == 0,
      [&](int64_t i, const float(&v)[W]) {
        if constexpr (OT != F64) {
          float y[W];
#pragma unroll
          for (int k = 0; k < W; ++k) y[k] = v[k] * coef;
          store_w<OT, W, true>(out, i, y);
        }
      },
      [&](int64_t i, auto v) {
        if constexpr (GT == F64 && OT == F64) reinterpret_cast<double*>(out)[i] = v * coef64;
        else if constexpr (GT == F64) put<OT>(out, i, (float)(v * coef64));
        else put<OT>(out, i, v * coef);
      });
}

template <int GT>
__device__ __forceinline__ void scale_run(int ot, const void* g, void* out, int64_t e0, int64_t e1,
                                          double coef) {
  switch (ot) {
    case F32: scale_run<GT, F32>(g, out, e0, e1, coef); break;
    case F16: scale_run<GT, F16>(g, out, e0, e1, coef); break;
    case BF16: scale_run<GT, BF16>(g, out, e0, e1, coef); break;
    default: scale_run<GT, F64>(g, out, e0, e1, coef); break;
  }
}

template <class T>
__device__ __forceinline__ void scale_runs(const T& rows, int count, uint32_t runs, int run,
                                           double coef) {
  for (uint32_t r = blockIdx.x; r < runs; r += gridDim.x) {
    const int t = tensor_of(rows, count, r);
    void* out = rows[t].out;
    if (!out) continue;
    const int64_t e0 = (int64_t)(r - rows[t].first) * run, e1 = min(rows[t].n, e0 + run);
    switch (rows[t].gt) {
      case F32: scale_run<F32>(rows[t].ot, rows[t].g, out, e0, e1, coef); break;
      case F16: scale_run<F16>(rows[t].ot, rows[t].g, out, e0, e1, coef); break;
      case BF16: scale_run<BF16>(rows[t].ot, rows[t].g, out, e0, e1, coef); break;
      default: scale_run<F64>(rows[t].ot, rows[t].g, out, e0, e1, coef); break;
    }
  }
}

template <bool TABLE>
__global__ __launch_bounds__(256) void norm_scale_kernel(const NormRows l,
                                                         const NormRow* __restrict__ table,
                                                         int count, uint32_t runs, int run,
                                                         const double* __restrict__ slots,
                                                         int nslots, double max_norm, double eps,
                                                         float* __restrict__ norm) {
  __shared__ double part[4];
  double s = 0.0;
  for (int i = threadIdx.x; i < nslots; i += 256) s += slots[i];
  const double nv = sqrt(block_sum(s, part));
  if (blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)nv;
  const double q = max_norm / (nv + eps), coef = q > 1.0 ? 1.0 : q;  // (NaN stays)
  if constexpr (TABLE) scale_runs(table, count, runs, run, coef);
  else scale_runs(l.row, count, runs, run, coef);
}

}  // namespace

size_t clip_grad_norm_workspace(int64_t count) {
  return BLOCKS * sizeof(double) + (count > ROWS ? (size_t)count * sizeof(NormRow) : 0);
}

int clip_grad_norm_launch(const novaq_gradient* list, int64_t count, double max_norm, double eps,
                          float* norm, void* workspace, hipStream_t st) {
  double* slots = static_cast<double*>(workspace);
  NormRow* table = reinterpret_cast<NormRow*>(slots + BLOCKS);
  int64_t total = 0, kept = 0;
  bool outputs = false;
  for (int64_t i = 0; i < count; ++i) {
    total += list[i].n;
    kept += list[i].n > 0;
    outputs |= list[i].out != nullptr && list[i].n > 0;
  }
  int64_t run = STEP;
  while (run < 8 * STEP && total / run > BLOCKS) run *= 2;
  int64_t runs = 0;
  for (int64_t i = 0; i < count; ++i) runs += (list[i].n + run - 1) / run;
  if (runs > 0x7FFFFFFF || kept > 0x7FFFFFFF) return NOVAQ_ENOTSUP;
  const bool by_table = kept > ROWS;
  NormRows l;
  int64_t at = 0, first = 0, done = 0;
  do {
    int k = 0;
    for (; at < count && k < ROWS; ++at) {
      const novaq_gradient& g = list[at];
      if (g.n == 0) continue;
      l.row[k++] = NormRow{g.grad, g.out, g.n, (uint32_t)first, (uint8_t)g.grad_dtype,
                           (uint8_t)g.out_dtype};
      first += (g.n + run - 1) / run;
    }
    if (by_table && k > 0) {
      hipLaunchKernelGGL(norm_rows_kernel, dim3(1), dim3(128), 0, st, l, k, table + done);
      const int rc = check_launch();
      if (rc != NOVAQ_OK) return rc;
      done += k;
    }
  } while (at < count);
  const int blocks = (int)std::min<int64_t>(runs, BLOCKS);
  const int scalers = std::max(1, outputs ? blocks : 1);
  if (blocks > 0) {
    if (by_table)
      hipLaunchKernelGGL(norm_sum_kernel<true>, dim3(blocks), dim3(256), 0, st, l, table,
                         (int)kept, (uint32_t)runs, (int)run, slots);
    else
      hipLaunchKernelGGL(norm_sum_kernel<false>, dim3(blocks), dim3(256), 0, st, l, table,
                         (int)kept, (uint32_t)runs, (int)run, slots);
    const int rc = check_launch();
    if (rc != NOVAQ_OK) return rc;
  }
  const uint32_t scaled = outputs ? (uint32_t)runs : 0u;
  if (by_table)
    hipLaunchKernelGGL(norm_scale_kernel<true>, dim3(scalers), dim3(256), 0, st, l, table,
                       (int)kept, scaled, (int)run, slots, blocks, max_norm, eps, norm);
  else
    hipLaunchKernelGGL(norm_scale_kernel<false>, dim3(scalers), dim3(256), 0, st, l, table,
                       (int)kept, scaled, (int)run, slots, blocks, max_norm, eps, norm);
  return check_launch();
}

}  // namespace novaq
