// Element access shared by the token kernels: rows of any stored type read 8
// elements at a time, ids of 32 or 64 bits.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "novaq_convert.h"

namespace novaq {
namespace {

typedef uint32_t ti_u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t ti_u32x4 __attribute__((ext_vector_type(4)));

// A token (or target) id: 32 or 64 bits, any value.
__device__ __forceinline__ int64_t token_at(const void* ids, int bits, int64_t i) {
  return bits == 64 ? reinterpret_cast<const int64_t*>(ids)[i]
                    : (int64_t) reinterpret_cast<const int32_t*>(ids)[i];
}

// Bytes of a stored row of D elements (E2M1 rows end on whole bytes).
__host__ __device__ inline int64_t row_bytes(int dtype, int64_t D) {
  return (D * dtype_bits(dtype) + 7) / 8;
}

// A vector load or store, past the caches where what it touches is not used
// again (NT; streams of hundreds of MB run half as fast again so).
template <bool NT, class T>
__device__ __forceinline__ T vload(const T* p) {
  if constexpr (NT) return __builtin_nontemporal_load(p);
  else return *p;
}
template <bool NT, class T>
__device__ __forceinline__ void vstore(T* p, const T& v) {
  if constexpr (NT) __builtin_nontemporal_store(v, p);
  else *p = v;
}

// Elements c .. c + 7 of a row of D as fp32 (zeros past D), c a multiple of
// 8.  VEC: D % 8 == 0 and the row starts on a boundary of 8 elements, so the
// run is one or two whole vector loads.
template <int ST, bool VEC, bool NT = false>
__device__ __forceinline__ void load8(const uint8_t* row, int64_t c, int64_t D, float (&v)[8]) {
  if constexpr (VEC) {
    if constexpr (ST == F32) {
      const ti_u32x4* p = reinterpret_cast<const ti_u32x4*>(row + c * 4);
      const ti_u32x4 a = vload<NT>(p), b = vload<NT>(p + 1);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = u2f(a[i]), v[4 + i] = u2f(b[i]);
    } else if constexpr (ST == F16 || ST == BF16) {
      const ti_u32x4 a = vload<NT>(reinterpret_cast<const ti_u32x4*>(row + c * 2));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t w = a[i];
        v[2 * i] = u2f(decode<ST>(w & 0xFFFFu));
        v[2 * i + 1] = u2f(decode<ST>(w >> 16));
      }
    } else if constexpr (ST == E4M3 || ST == E5M2) {
      const ti_u32x2 a = vload<NT>(reinterpret_cast<const ti_u32x2*>(row + c));
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t w = a[i >> 2];
        v[i] = u2f(decode<ST>((w >> (8 * (i & 3))) & 0xFFu));
      }
    } else {
      const uint32_t w = vload<NT>(reinterpret_cast<const uint32_t*>(row + c / 2));
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = u2f(decode<E2M1>((w >> (4 * i)) & 0xFu));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t e = c + i;
      uint32_t code = 0;
      if (e < D) {
        if constexpr (ST == F32) code = reinterpret_cast<const uint32_t*>(row)[e];
        else if constexpr (ST == F16 || ST == BF16)
          code = reinterpret_cast<const uint16_t*>(row)[e];
        else if constexpr (ST == E2M1) code = (row[e >> 1] >> (4 * (e & 1))) & 0xFu;
        else code = row[e];
      }
      v[i] = u2f(decode<ST>(code));
    }
  }
}

// 8 fp32 values stored as OT (F32, F16, BF16) at element e of out; whole
// vectors (VEC: e on a boundary of 8 and 16-byte aligned) or the first `left`.
template <int OT, bool VEC, bool NT = false>
__device__ __forceinline__ void store8(void* out, int64_t e, int64_t left, const float (&v)[8]) {
  if constexpr (OT == F32) {
    float* p = reinterpret_cast<float*>(out) + e;
    if constexpr (VEC) {
      ti_u32x4 a, b;
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = f2u(v[i]), b[i] = f2u(v[4 + i]);
      vstore<NT>(reinterpret_cast<ti_u32x4*>(p), a);
      vstore<NT>(reinterpret_cast<ti_u32x4*>(p) + 1, b);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < left) p[i] = v[i];
    }
  } else {
    uint16_t* p = reinterpret_cast<uint16_t*>(out) + e;
    if constexpr (VEC) {
      ti_u32x4 a;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (OT == BF16) a[i] = pack_bf16x2(f2u(v[2 * i]), f2u(v[2 * i + 1]));
        else a[i] = encode<F16>(f2u(v[2 * i])) | (encode<F16>(f2u(v[2 * i + 1])) << 16);
      }
      vstore<NT>(reinterpret_cast<ti_u32x4*>(p), a);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < left) p[i] = (uint16_t)encode<OT>(f2u(v[i]));
    }
  }
}

}  // namespace
}  // namespace novaq
