// Clipping of many gradients by their global norm.
//
//   norm = sqrt(sum over all tensors and elements of g^2)
//   out  = g * min(1, max_norm / (norm + eps))
//
// Two passes over memory: the first leaves one fp64 sum of squares a workgroup
// (products and sums in fp64, so neither the largest fp32 gradient nor the
// smallest one leaves the range), the second adds these in a fixed order in
// every workgroup (from L2) and scales.  The tensors' addresses and lengths
// travel in the kernels' arguments, 96 tensors a launch: nothing is copied to
// the device and nothing about a tensor outlives the call.  Workgroups walk
// runs of 4096 elements of one launch's tensors.
//
// NaN or infinite gradients give a NaN or infinite norm: the factor is then
// NaN or 0, as the formula says (min keeps a NaN).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "novaq_internal.h"
#include "token_io.h"

namespace novaq {
namespace {

constexpr int F64 = NOVAQ_F64;     // (only here: float64 gradients)
constexpr int TENSORS = 96;        // a launch: 3 KB of kernel arguments
constexpr int RUN = 4096;          // elements of one workgroup's step
constexpr int SLOTS = 2048;        // workgroups (and fp64 sums) over all launches

struct NormList {
  const void* g[TENSORS];
  void* out[TENSORS];
  int64_t n[TENSORS];
  uint32_t first[TENSORS];  // its first run among the launch's
  uint8_t gt[TENSORS], ot[TENSORS];
  int count;
  uint32_t runs;
};

// The tensor that holds run r of the list.
__device__ __forceinline__ int tensor_of(const NormList& l, uint32_t r) {
  int lo = 0, hi = l.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (l.first[mid] <= r) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ double block_sum(double s, double* part) {
#pragma unroll
  for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  s = part[0];
  for (int w = 1; w < (int)blockDim.x / 64; ++w) s += part[w];
  __syncthreads();
  return s;
}

// f(i, v, m): m (1 or V) values from element i on, over the run at e0.
template <int GT, class F>
__device__ __forceinline__ void each_of_run(const void* p, int64_t n, int64_t e0, F&& f) {
  const int64_t e1 = min(n, e0 + RUN);
  const uint8_t* b = static_cast<const uint8_t*>(p);
  if constexpr (GT == F64) {
    for (int64_t i = e0 + threadIdx.x; i < e1; i += blockDim.x) {
      const double v[1] = {reinterpret_cast<const double*>(b)[i]};
      f(i, v, 1);
    }
  } else {
    const bool vec = (reinterpret_cast<uintptr_t>(b) & 15) == 0;
    const int64_t whole = vec ? e0 + (e1 - e0) / 8 * 8 : e0;
#pragma unroll 2
    for (int64_t i = e0 + threadIdx.x * 8; i < whole; i += blockDim.x * 8) {
      float v[8];
      load8<GT, true>(b, i, n, v);
      f(i, v, 8);
    }
    for (int64_t i = whole + threadIdx.x; i < e1; i += blockDim.x) {
      float v[1];
      if constexpr (GT == F32) v[0] = reinterpret_cast<const float*>(b)[i];
      else v[0] = u2f(decode<GT>(reinterpret_cast<const uint16_t*>(b)[i]));
      f(i, v, 1);
    }
  }
}

__global__ __launch_bounds__(256) void norm_sum_kernel(const NormList l,
                                                       double* __restrict__ slots) {
  __shared__ double part[4];
  double s = 0.0;
  auto add = [&](int64_t, const auto* v, int m) {
    for (int i = 0; i < m; ++i) {
      const double d = (double)v[i];
      s = fma(d, d, s);
    }
  };
  for (uint32_t r = blockIdx.x; r < l.runs; r += gridDim.x) {
    const int t = tensor_of(l, r);
    const int64_t e0 = (int64_t)(r - l.first[t]) * RUN;
    switch (l.gt[t]) {
      case F32: each_of_run<F32>(l.g[t], l.n[t], e0, add); break;
      case F16: each_of_run<F16>(l.g[t], l.n[t], e0, add); break;
      case BF16: each_of_run<BF16>(l.g[t], l.n[t], e0, add); break;
      default: each_of_run<F64>(l.g[t], l.n[t], e0, add); break;
    }
  }
  s = block_sum(s, part);
  if (threadIdx.x == 0) slots[blockIdx.x] = s;
}

__device__ __forceinline__ void put(void* out, int ot, int64_t i, double v) {
  switch (ot) {
    case F32: reinterpret_cast<float*>(out)[i] = (float)v; break;
    case F16: reinterpret_cast<uint16_t*>(out)[i] = (uint16_t)encode<F16>(f2u((float)v)); break;
    case BF16: reinterpret_cast<uint16_t*>(out)[i] = (uint16_t)encode<BF16>(f2u((float)v)); break;
    default: reinterpret_cast<double*>(out)[i] = v; break;
  }
}

__global__ __launch_bounds__(256) void norm_scale_kernel(const NormList l,
                                                         const double* __restrict__ slots,
                                                         int nslots, float max_norm, float eps,
                                                         float* __restrict__ norm) {
  __shared__ double part[4];
  double s = 0.0;
  for (int i = threadIdx.x; i < nslots; i += 256) s += slots[i];
  s = block_sum(s, part);
  const float nv = (float)sqrt(s);
  if (blockIdx.x == 0 && threadIdx.x == 0) *norm = nv;
  const float q = max_norm / (nv + eps), coef = q > 1.0f ? 1.0f : q;  // (NaN stays)
  for (uint32_t r = blockIdx.x; r < l.runs; r += gridDim.x) {
    const int t = tensor_of(l, r);
    if (!l.out[t]) continue;
    const int64_t e0 = (int64_t)(r - l.first[t]) * RUN;
    void* out = l.out[t];
    const int ot = l.ot[t];
    const bool vec = (reinterpret_cast<uintptr_t>(out) & 15) == 0;
    auto scale = [&](int64_t i, const auto* v, int m) {
      if (m == 8) {
        float y[8];
        for (int k = 0; k < 8; ++k) y[k] = (float)v[k] * coef;
        if (vec && ot == F32) store8<F32, true>(out, i, 8, y);
        else if (vec && ot == F16) store8<F16, true>(out, i, 8, y);
        else if (vec && ot == BF16) store8<BF16, true>(out, i, 8, y);
        else
          for (int k = 0; k < 8; ++k) put(out, ot, i + k, (double)y[k]);
      } else if constexpr (sizeof(v[0]) == 8) {
        put(out, ot, i, v[0] * (double)coef);
      } else {
        put(out, ot, i, (double)(v[0] * coef));
      }
    };
    switch (l.gt[t]) {
      case F32: each_of_run<F32>(l.g[t], l.n[t], e0, scale); break;
      case F16: each_of_run<F16>(l.g[t], l.n[t], e0, scale); break;
      case BF16: each_of_run<BF16>(l.g[t], l.n[t], e0, scale); break;
      default: each_of_run<F64>(l.g[t], l.n[t], e0, scale); break;
    }
  }
}

}  // namespace

size_t clip_grad_norm_workspace(int64_t count) {
  // one slot a workgroup; launches of at most SLOTS over all of them, at least
  // one workgroup each
  return (size_t)(SLOTS + (count + TENSORS - 1) / TENSORS) * 8;
}

int clip_grad_norm_launch(const novaq_gradient* list, int64_t count, float max_norm, float eps,
                          float* norm, void* workspace, hipStream_t st) {
  double* slots = static_cast<double*>(workspace);
  int64_t total = 0;
  bool outputs = false;
  for (int64_t i = 0; i < count; ++i) {
    total += (list[i].n + RUN - 1) / RUN;
    outputs |= list[i].out != nullptr && list[i].n > 0;
  }
  int used = 0;
  for (int pass = 0; pass < 2; ++pass) {
    int64_t at = 0;
    bool first = true;
    do {
      NormList l;
      l.count = 0;
      int64_t runs = 0;
      while (at < count && l.count < TENSORS) {
        const novaq_gradient& g = list[at];
        const int64_t r = (g.n + RUN - 1) / RUN;
        if (runs + r > 0x7FFFFFFF && l.count) break;
        ++at;
        if (g.n == 0) continue;
        l.g[l.count] = g.grad;
        l.out[l.count] = g.out;
        l.n[l.count] = g.n;
        l.gt[l.count] = (uint8_t)g.grad_dtype;
        l.ot[l.count] = (uint8_t)g.out_dtype;
        l.first[l.count++] = (uint32_t)runs;
        runs += r;
      }
      l.runs = (uint32_t)runs;
      if (runs == 0 && !(pass == 1 && first)) continue;
      if (pass == 0) {
        const int blocks = (int)std::max<int64_t>(1, std::min(runs, runs * SLOTS / total));
        hipLaunchKernelGGL(norm_sum_kernel, dim3(blocks), dim3(256), 0, st, l, slots + used);
        used += blocks;
      } else {
        const int blocks = (int)std::max<int64_t>(1, outputs ? std::min<int64_t>(runs, SLOTS) : 1);
        hipLaunchKernelGGL(norm_scale_kernel, dim3(blocks), dim3(256), 0, st, l, slots, used,
                           max_norm, eps, norm);
      }
      first = false;
      const int rc = check_launch();
      if (rc != NOVAQ_OK) return rc;
      if (pass == 1 && !outputs) return NOVAQ_OK;  // the norm is all that is asked for
    } while (at < count);
  }
  return NOVAQ_OK;
}

}  // namespace novaq
