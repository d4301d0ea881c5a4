// The AdamW step of many tensors at once, for gfx950: fp32 weights, gradients of any
// float type, states in fp32 or in 8 bits, and the FP8 codes that weights keep beside.
//
//   m = b1 m + (1 - b1) g;   v = b2 v + (1 - b2) g^2
//   w = w - (lr (m / bc1)) / (sqrt(v / bc2) + eps);   w = w - (lr wd) w   (where it decays)
//
// each a float32 operation in this order, so that fp32 states give the bits of the step
// of one tensor (optim.hip).
//
// States in 8 bits: 128 elements in a row share an exponent e (a scale of 2^(e - 127)) for
// m and one for v.
//   m is E4M3 with the smallest scale that holds the block's largest.
//   v has no sign: code c > 0 is the float with the bits (c << 20) + ((e - 31) << 23), 5
//     bits of exponent and 3 of mantissa below the block's largest; 0 is 0.
// A step moves v by a thousandth of its distance to g^2, much less than half a code, so
// rounding to nearest would leave it where it is.  Both are rounded at random instead, up
// with the probability of their place between two codes: then the mean of the codes is
// the fp32 recurrence.  What that costs is a relative deviation of v of about a tenth of a
// code a step, summed over 1 / (1 - b2) steps.  A v that is not zero never becomes zero: m
// could otherwise meet a denominator of eps.  The random numbers are a hash of the
// element's place and a key from the step's seed: the same call gives the same bits, and
// no state is kept.  A block with an infinity or a NaN has the exponent 255 and decodes to
// NaN from then on.
//
// Bound by memory: w is read and written (8 bytes), the gradient read (2 or 4), and the
// states read and written (16 bytes, or 4).  A launch takes 48 tensors, whose addresses
// travel in its arguments: they are cut into runs, one a workgroup, each looked up by
// bisection in the tensors' first runs.  4 consecutive elements a lane: every load of a wave
// covers whole lines.  Weights with FP8 blocks are stepped a tile of 128 x 128 a workgroup
// where that pays, which then has their codes' scale.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "block_quant.h"

namespace novaq {
namespace {

typedef float am_f32x4 __attribute__((ext_vector_type(4)));
typedef float am_f32x2 __attribute__((ext_vector_type(2)));

struct StepRow {
  float* w;
  const void* g;
  void *m, *v;
  uint8_t *me, *ve;  // null: fp32 states
  uint32_t* amax;    // gets max |w| (NaN passed over), or null
  int64_t n;
  uint32_t first;    // its first run
  uint32_t base;     // the place of its first element in the list's random numbers
  uint8_t gt, decay, s8, vec;
};
static_assert(sizeof(StepRow) == 80, "48 rows fit a kernel's arguments");
constexpr int STEP_ROWS = 48;
struct StepRows {
  StepRow row[STEP_ROWS];
};

// A weight with FP8 blocks, a tile of 128 x 128 a workgroup.
struct TileRow {
  float* w;
  const void* g;
  void *m, *v;
  uint8_t *me, *ve;
  BlockOut o;
  int32_t R, C;
  uint32_t first;  // its first tile
  uint32_t base;
  uint8_t gt, decay, s8, dt;
};
static_assert(sizeof(TileRow) == 104, "32 rows fit a kernel's arguments");
constexpr int TILE_ROWS = 32;
struct TileRows {
  TileRow row[TILE_ROWS];
};

// The scalars as numpy rounds them (optim.hip), and for 8-bit states lr / bc1 and
// 1 / sqrt(bc2).
struct StepHP {
  float b1, omb1, b2, omb2, bc1, bc2, lr, eps, lrwd, lr_m, root_v;
};

// A run: what a workgroup has, 4 elements a lane, or twice that in 8 bits.  One run a
// workgroup: with 2048 workgroups that took runs in turn 8-bit states of 336 M elements took
// 1024 us, so 914 (4 elements a lane 944), fp32 states 1770, so 1596 (8 a lane 1670).
__host__ __device__ constexpr int step_run_length(bool s8) { return s8 ? 2048 : 1024; }

__global__ __launch_bounds__(64) void step_clear_kernel(const StepRows l, int count) {
  const int i = threadIdx.x;
  if (i < count && l.row[i].amax) *l.row[i].amax = 0u;
}

template <class T>
__device__ __forceinline__ int row_of(const T& rows, int count, uint32_t r) {
  int lo = 0, hi = count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (rows[mid].first <= r) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// FAST: the hardware's root and reciprocal (1 unit in the last place each, 2^-23) and constants
// multiplied beforehand (two, rounded once: 2^-24 each), with four products and sums rounded
// once: such a step is within 10 * 2^-24 < 2^-20 of itself, far below a rounding of w;
// correctly rounded ones are a third of the instructions that bound 8-bit states (336 M
// elements with bf16 gradients 1182 us with them, 1024 with the hardware's).
template <bool FAST>
__device__ __forceinline__ float step_element(float w, float g, float& m, float& v,
                                              const StepHP& h, bool decay) {
  m = h.b1 * m + h.omb1 * g;
  v = h.b2 * v + h.omb2 * (g * g);
  if constexpr (FAST) {
    const float root = __builtin_amdgcn_sqrtf(v) * h.root_v + h.eps;
    w = w - (h.lr_m * m) * __builtin_amdgcn_rcpf(root);
    return decay ? w - h.lrwd * w : w;
  }
  const float m_hat = m / h.bc1;
  const float v_hat = v / h.bc2;
  w = w - (h.lr * m_hat) / (sqrtf(v_hat) + h.eps);
  return decay ? w - h.lrwd * w : w;
}

// A 32-bit random number of an element: multiplications by the fractional parts of the
// golden ratio and of the square root of 2, with its halves folded between.
__device__ __forceinline__ uint32_t step_random(uint32_t element, uint32_t key) {
  uint32_t h = (element + key) * 0x9E3779B9u;
  h = (h ^ (h >> 16)) * 0x6A09E667u;
  return h ^ (h >> 15);
}

// max over the 32 lanes that hold a block, in all of them.
__device__ __forceinline__ uint32_t max32(uint32_t a) {
  a = bq_max16(a);
  return max(a, (uint32_t)__shfl_xor((int)a, 16));
}

__device__ __forceinline__ int m_exponent(uint32_t top) {
  const int e = (int)(top >> 23) - 8 + ((top & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return top >= 0x7F800000u ? 255 : max(e, 1);
}
__device__ __forceinline__ int v_exponent(uint32_t top) {
  const int e = (int)(top >> 23) + ((top & 0x7FFFFFu) > 0x700000u ? 1 : 0);
  return top >= 0x7F800000u ? 255 : min(max(e, 40), 254);
}
// (255 is NaN, whatever the code)
__device__ __forceinline__ float m_scale(int e) { return e == 255 ? u2f(0x7FC00000u) : bq_scale(e); }
__device__ __forceinline__ float v_value(uint32_t c, int e) {
  const uint32_t nan = e == 255 ? 0x7FC00000u : 0u;
  return u2f(nan | (c ? (c << 20) + ((uint32_t)(e - 31) << 23) : 0u));
}

__device__ __forceinline__ void m_values(uint32_t codes, float s, float (&m)[4]) {
  const am_f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, false);
  const am_f32x2 b = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, true);
  m[0] = a[0] * s, m[1] = a[1] * s, m[2] = b[0] * s, m[3] = b[1] * s;
}

// m's code: |m| / scale (exact) is at most 448.  Normal codes from 2^-6: the 20 bits of the
// mantissa that fall away, and 20 random ones, carry; below, in units of 2^-9.
__device__ __forceinline__ uint32_t m_code(float m, float inv, uint32_t random) {
  const float a = fabsf(m) * inv;
  const uint32_t normal = ((f2u(a) + random) >> 20) - (120u << 3);
  const uint32_t small = (uint32_t)(a * 512.0f + (float)random * 0x1p-20f);
  return (a < 0x1p-6f ? small : normal) | (f2u(m) >> 24 & 0x80u);
}
__device__ __forceinline__ uint32_t v_code(float v, int e, uint32_t random) {
  const int32_t c = (int32_t)(f2u(v) - ((uint32_t)(e - 31) << 23));
  const uint32_t up = c < (1 << 20) ? 1u : min((uint32_t)(c + (int32_t)random) >> 20, 255u);
  return v > 0.0f ? up : 0u;
}

// 4 elements from i on (fewer at a tensor's end: zeros), as fp32.  NT: past the caches.
template <int GT, bool NT>
__device__ __forceinline__ void load4(const void* p, int64_t i, int64_t n, bool vec,
                                      float (&v)[4]) {
  if (vec && i + 4 <= n) {
    if constexpr (GT == F32) {
      const am_f32x4 a =
          vload<NT>(reinterpret_cast<const am_f32x4*>(static_cast<const float*>(p) + i));
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = a[k];
    } else {
      const ti_u32x2 a =
          vload<NT>(reinterpret_cast<const ti_u32x2*>(static_cast<const uint16_t*>(p) + i));
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = bq_value16<GT>(a[k >> 1] >> (16 * (k & 1)) & 0xFFFFu);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[k] = 0.0f;
      if (i + k < n) {
        if constexpr (GT == F32) v[k] = static_cast<const float*>(p)[i + k];
        else v[k] = bq_value16<GT>(static_cast<const uint16_t*>(p)[i + k]);
      }
    }
  }
}
template <bool NT>
__device__ __forceinline__ void store4(void* p, int64_t i, int64_t n, bool vec,
                                       const float (&v)[4]) {
  float* to = static_cast<float*>(p) + i;
  if (vec && i + 4 <= n) {
    vstore<NT>(reinterpret_cast<am_f32x4*>(to), am_f32x4{v[0], v[1], v[2], v[3]});
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (i + k < n) to[k] = v[k];
  }
}
template <bool NT>
__device__ __forceinline__ uint32_t load_codes(const void* p, int64_t i, int64_t n, bool vec) {
  const uint8_t* at = static_cast<const uint8_t*>(p) + i;
  if (vec && i + 4 <= n) return vload<NT>(reinterpret_cast<const uint32_t*>(at));
  uint32_t w = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (i + k < n) w |= (uint32_t)at[k] << (8 * k);
  return w;
}
template <bool NT>
__device__ __forceinline__ void store_codes(void* p, int64_t i, int64_t n, bool vec, uint32_t w) {
  uint8_t* at = static_cast<uint8_t*>(p) + i;
  if (vec && i + 4 <= n) {
    vstore<NT>(reinterpret_cast<uint32_t*>(at), w);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (i + k < n) at[k] = (uint8_t)(w >> (8 * k));
  }
}

// One run of a tensor, from element s0 on; its largest |w| where that is asked for.
template <int GT, bool S8, bool NT>
__device__ __forceinline__ uint32_t step_run(const StepRow& t, int64_t s0, const StepHP& h,
                                             uint32_t key) {
  constexpr int STEP_UNROLL = step_run_length(S8) / 1024;
  const bool vec = t.vec, decay = t.decay;
  const int64_t n = t.n;
  uint32_t top = 0;
  float w[STEP_UNROLL][4], g[STEP_UNROLL][4], m[STEP_UNROLL][4], v[STEP_UNROLL][4];
  uint32_t mc[STEP_UNROLL], vc[STEP_UNROLL];
  int me[STEP_UNROLL], ve[STEP_UNROLL];
  // (lanes past the tensor's end hold zeros)
#pragma unroll
  for (int u = 0; u < STEP_UNROLL; ++u) {
    const int64_t i = s0 + u * 1024 + threadIdx.x * 4;
    load4<F32, NT>(t.w, i, n, vec, w[u]);
    load4<GT, NT>(t.g, i, n, vec, g[u]);
    if constexpr (S8) {
      mc[u] = load_codes<NT>(t.m, i, n, vec);
      vc[u] = load_codes<NT>(t.v, i, n, vec);
      me[u] = i < n ? t.me[i >> 7] : 0;
      ve[u] = i < n ? t.ve[i >> 7] : 0;
    } else {
      load4<F32, NT>(t.m, i, n, vec, m[u]);
      load4<F32, NT>(t.v, i, n, vec, v[u]);
    }
  }
#pragma unroll
  for (int u = 0; u < STEP_UNROLL; ++u) {
    const int64_t i = s0 + u * 1024 + threadIdx.x * 4;
    if constexpr (S8) {
      m_values(mc[u], m_scale(me[u]), m[u]);
#pragma unroll
      for (int k = 0; k < 4; ++k) v[u][k] = v_value(vc[u] >> (8 * k) & 0xFFu, ve[u]);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) w[u][k] = step_element<S8>(w[u][k], g[u][k], m[u][k], v[u][k], h, decay);
    if (t.amax) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (i + k < n) top = max(top, bq_mag_number(w[u][k]));
    }
    store4<NT>(t.w, i, n, vec, w[u]);
    if constexpr (S8) {
      uint32_t tm = 0, tv = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        tm = max(tm, i + k < n ? bq_mag(m[u][k]) : 0u);
        tv = max(tv, i + k < n ? bq_mag(v[u][k]) : 0u);
      }
      const int xm = m_exponent(max32(tm)), xv = v_exponent(max32(tv));
      // (255: no code matters)
      const float inv = bq_inverse(xm);
      uint32_t cm = 0, cv = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t r = step_random(t.base + (uint32_t)(i + k), key);
        cm |= m_code(m[u][k], inv, (r >> 16) << 4 | 8u) << (8 * k);
        cv |= v_code(v[u][k], xv, (r & 0xFFFFu) << 4 | 8u) << (8 * k);
      }
      store_codes<NT>(t.m, i, n, vec, xm == 255 ? 0u : cm);
      store_codes<NT>(t.v, i, n, vec, xv == 255 ? 0u : cv);
      if ((threadIdx.x & 31) == 0 && i < n) {
        t.me[i >> 7] = (uint8_t)xm;
        t.ve[i >> 7] = (uint8_t)xv;
      }
    } else {
      store4<NT>(t.m, i, n, vec, m[u]);
      store4<NT>(t.v, i, n, vec, v[u]);
    }
  }
  return top;
}

// NT: the tensors of the step are more than the 256 MB that the last cache holds (336 M
// elements with 8-bit states 852 us, through the caches 891; with fp32 states 1542 and 1593;
// 10 M with 8-bit states, which it holds, 32.1 and 30.7).
template <bool NT>
__global__ __launch_bounds__(256) void step_kernel(const StepRows l, int count, uint32_t runs,
                                                   const StepHP h, uint32_t key) {
  __shared__ uint32_t part[4];
  for (uint32_t r = blockIdx.x; r < runs; r += gridDim.x) {
    const StepRow& t = l.row[row_of(l.row, count, r)];
    const int64_t s0 = (int64_t)(r - t.first) * step_run_length(t.s8);
    uint32_t top;
    if (t.s8) {
      if (t.gt == F32) top = step_run<F32, true, NT>(t, s0, h, key);
      else if (t.gt == F16) top = step_run<F16, true, NT>(t, s0, h, key);
      else top = step_run<BF16, true, NT>(t, s0, h, key);
    } else {
      if (t.gt == F32) top = step_run<F32, false, NT>(t, s0, h, key);
      else if (t.gt == F16) top = step_run<F16, false, NT>(t, s0, h, key);
      else top = step_run<BF16, false, NT>(t, s0, h, key);
    }
    if (t.amax) {
#pragma unroll
      for (int d = 32; d; d >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d));
      if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
      __syncthreads();
      if (threadIdx.x == 0) {
        top = max(max(part[0], part[1]), max(part[2], part[3]));
        // (the largest whatever their order; most need not wait for one another)
        if (top > __atomic_load_n(t.amax, __ATOMIC_RELAXED)) atomicMax(t.amax, top);
      }
      __syncthreads();
    }
  }
}

// The step of 8 elements of a row at element i, which are in the tensor and aligned: their
// states and w in memory, w here.
template <int GT, bool S8>
struct Step8 {
  Raw8<F32> w;
  Raw8<GT> g;
  typename std::conditional<S8, ti_u32x2, Raw8<F32>>::type m, v;
  uint32_t me, ve;
};
template <int GT, bool S8>
__device__ __forceinline__ void step8_load(const TileRow& t, int64_t i, Step8<GT, S8>& e) {
  e.w = raw8<F32, true>(t.w, 0, i, INT64_MAX);
  e.g = raw8<GT, true>(t.g, 0, i, INT64_MAX);
  if constexpr (S8) {
    e.m = *reinterpret_cast<const ti_u32x2*>(static_cast<const uint8_t*>(t.m) + i);
    e.v = *reinterpret_cast<const ti_u32x2*>(static_cast<const uint8_t*>(t.v) + i);
    e.me = t.me[i >> 7];
    e.ve = t.ve[i >> 7];
  } else {
    e.m = raw8<F32, true>(t.m, 0, i, INT64_MAX);
    e.v = raw8<F32, true>(t.v, 0, i, INT64_MAX);
  }
}
__device__ __forceinline__ void put8(void* p, int64_t i, const float (&v)[8]) {
  am_f32x4* to = reinterpret_cast<am_f32x4*>(static_cast<float*>(p) + i);
  to[0] = am_f32x4{v[0], v[1], v[2], v[3]};
  to[1] = am_f32x4{v[4], v[5], v[6], v[7]};
}
template <int GT, bool S8>
__device__ __forceinline__ void step8(const TileRow& t, int64_t i, const Step8<GT, S8>& e,
                                      const StepHP& h, uint32_t key, float (&w)[8]) {
  float g[8], m[8], v[8];
  values8<F32>(e.w, w);
  values8<GT>(e.g, g);
  if constexpr (S8) {
    float f[4];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      m_values(e.m[q], m_scale((int)e.me), f);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        m[4 * q + k] = f[k];
        v[4 * q + k] = v_value(e.v[q] >> (8 * k) & 0xFFu, (int)e.ve);
      }
    }
  } else {
    values8<F32>(e.m, m);
    values8<F32>(e.v, v);
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) w[k] = step_element<S8>(w[k], g[k], m[k], v[k], h, t.decay);
  put8(t.w, i, w);
  if constexpr (S8) {
    uint32_t tm = 0, tv = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) tm = max(tm, bq_mag(m[k])), tv = max(tv, bq_mag(v[k]));
    const int xm = m_exponent(bq_max16(tm)), xv = v_exponent(bq_max16(tv));
    const float inv = bq_inverse(xm);
    ti_u32x2 cm{0, 0}, cv{0, 0};
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t r = step_random(t.base + (uint32_t)i + k, key);
      cm[k >> 2] |= m_code(m[k], inv, (r >> 16) << 4 | 8u) << (8 * (k & 3));
      cv[k >> 2] |= v_code(v[k], xv, (r & 0xFFFFu) << 4 | 8u) << (8 * (k & 3));
    }
    if (xm == 255) cm = ti_u32x2{0, 0};
    if (xv == 255) cv = ti_u32x2{0, 0};
    *reinterpret_cast<ti_u32x2*>(static_cast<uint8_t*>(t.m) + i) = cm;
    *reinterpret_cast<ti_u32x2*>(static_cast<uint8_t*>(t.v) + i) = cv;
    if ((threadIdx.x & 15) == 0) {
      t.me[i >> 7] = (uint8_t)xm;
      t.ve[i >> 7] = (uint8_t)xv;
    }
  } else {
    put8(t.m, i, m);
    put8(t.v, i, v);
  }
}

// A thread's 4 x 8 elements of a tile (the blocks' own layout), zeros past the matrix.  Rows
// are fetched ahead, as many as 128 registers hold (8 weights of 4096 x 4096 8-bit states: all
// four 471 us, two 483; with 80 registers three workgroups fit a CU and spill).
template <int GT, bool S8>
__device__ __forceinline__ void step_tile(const TileRow& t, int64_t rt, int64_t ct,
                                          const StepHP& h, uint32_t key, float (&w)[BQ_R][8]) {
  const int64_t r0 = rt * BQ + (threadIdx.x >> 4) * BQ_R, c0 = ct * BQ + (threadIdx.x & 15) * 8;
  constexpr int AHEAD = S8 ? 4 : 2;
  Step8<GT, S8> e[AHEAD];
  auto in = [&](int i) { return r0 + i < t.R && c0 < t.C; };
#pragma unroll
  for (int i = 0; i < AHEAD; ++i)
    if (in(i)) step8_load<GT, S8>(t, (r0 + i) * t.C + c0, e[i]);
#pragma unroll
  for (int i = 0; i < BQ_R; ++i) {
#pragma unroll
    for (int k = 0; k < 8; ++k) w[i][k] = 0.0f;
    if (in(i)) step8<GT, S8>(t, (r0 + i) * t.C + c0, e[i % AHEAD], h, key, w[i]);
    if (i + AHEAD < BQ_R && in(i + AHEAD))
      step8_load<GT, S8>(t, (r0 + i + AHEAD) * t.C + c0, e[i % AHEAD]);
  }
}

__global__ __launch_bounds__(BQ_THREADS, 4) void step_tile_kernel(const TileRows l, int count,
                                                                  const StepHP h, uint32_t key) {
  __shared__ __attribute__((aligned(16))) BlockTileLds lds;
  const TileRow& t = l.row[row_of(l.row, count, blockIdx.x)];
  const int tile = (int)(blockIdx.x - t.first), ctiles = (t.C + 127) / 128;
  const int rt = tile / ctiles, ct = tile % ctiles;
  float w[BQ_R][8];
  if (t.s8) {
    if (t.gt == F32) step_tile<F32, true>(t, rt, ct, h, key, w);
    else if (t.gt == F16) step_tile<F16, true>(t, rt, ct, h, key, w);
    else step_tile<BF16, true>(t, rt, ct, h, key, w);
  } else {
    if (t.gt == F32) step_tile<F32, false>(t, rt, ct, h, key, w);
    else if (t.gt == F16) step_tile<F16, false>(t, rt, ct, h, key, w);
    else step_tile<BF16, false>(t, rt, ct, h, key, w);
  }
  if (t.dt == E4M3) bq_tile<E4M3, true>(w, t.R, t.C, rt, ct, t.o, nullptr, lds);
  else bq_tile<E5M2, true>(w, t.R, t.C, rt, ct, t.o, nullptr, lds);
}

// The FP8 blocks of weights that took their step in runs.
template <int DT>
__global__ __launch_bounds__(BQ_THREADS, 6) void step_blocks_kernel(const TileRows l, int count) {
  __shared__ __attribute__((aligned(16))) BlockTileLds lds;
  const TileRow& t = l.row[row_of(l.row, count, blockIdx.x)];
  const int tile = (int)(blockIdx.x - t.first), ctiles = (t.C + 127) / 128;
  const int rt = tile / ctiles, ct = tile % ctiles;
  float v[BQ_R][8];
  bq_load<F32, false>(t.w, t.R, t.C, rt, ct, v);
  bq_tile<DT, true>(v, t.R, t.C, rt, ct, t.o, nullptr, lds);
}

template <int OT>
__global__ __launch_bounds__(256) void state_decode_kernel(const uint8_t* __restrict__ m,
                                                           const uint8_t* __restrict__ me,
                                                           const uint8_t* __restrict__ v,
                                                           const uint8_t* __restrict__ ve,
                                                           int64_t n, void* __restrict__ om,
                                                           void* __restrict__ ov, bool vec) {
  const int64_t stride = (int64_t)gridDim.x * 2048;
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8; i < n; i += stride) {
    const float sm = m_scale(me[i >> 7]);
    const int xv = ve[i >> 7];
    float a[8], b[8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t mc = load_codes<false>(m, i + 4 * h, n, vec);
      const uint32_t vc = load_codes<false>(v, i + 4 * h, n, vec);
      float f[4];
      m_values(mc, sm, f);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        a[4 * h + k] = f[k];
        b[4 * h + k] = v_value(vc >> (8 * k) & 0xFFu, xv);
      }
    }
    if (vec && i + 8 <= n) {
      if (om) store8<OT, true, true>(om, i, 8, a);
      if (ov) store8<OT, true, true>(ov, i, 8, b);
    } else {
      if (om) store8<OT, false>(om, i, n - i, a);
      if (ov) store8<OT, false>(ov, i, n - i, b);
    }
  }
}

bool on(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

uint32_t tiles_of(const TileRow& t) {
  return (uint32_t)((t.R + 127) / 128) * (uint32_t)((t.C + 127) / 128);
}

// Whether a weight with blocks may take its step tile by tile, w then read once: a tile's
// rows need whole accesses of 8 elements, and 8-bit states blocks that lie in its rows.
// Others are stepped in runs and their tiles read again.
bool fits_tiles(const novaq_adamw_tensor& t) {
  if (!t.codes || t.amax_scale || t.n == 0) return false;
  const bool s8 = t.m_exponents != nullptr;
  const uintptr_t sa = s8 ? 8 : 16;
  return t.cols % (s8 ? 128 : 8) == 0 && on(t.w, 16) && on(t.grad, 16) && on(t.m, sa) &&
         on(t.v, sa);
}

// Whether a per-tensor weight is stepped by the kernel of one tensor (optim.hip): the large one
// of a call.  Its 2048 workgroups join their largest |w| in its amax once each, a list's one for
// each run (E4M3 codes and fp32 gradients, the cast with it: 4096 x 4096 97 us so, 115 in the
// list; 2048 x 2048 50 and 55; 1024 x 1024 24 both ways).  Several large ones take a launch or
// two more each so (4 of 2048 x 2048 175 us, in the list 133; 4 of 4096 x 4096 410 and 413).
bool steps_alone(const novaq_adamw_tensor& t, int64_t elements) {
  return t.amax_scale && !t.m_exponents && t.grad_dtype == F32 && t.n >= (1 << 22) &&
         t.n > elements / 2 && on(t.w, 16) && on(t.grad, 16) && on(t.m, 16) && on(t.v, 16);
}

}  // namespace

int adamw_many_launch(const novaq_adamw_tensor* list, int64_t count, const novaq_adamw& hp,
                      uint32_t key, hipStream_t st) {
  StepHP h;
  h.b1 = (float)hp.beta1;
  h.omb1 = (float)(1.0 - hp.beta1);
  h.b2 = (float)hp.beta2;
  h.omb2 = (float)(1.0 - hp.beta2);
  h.bc1 = (float)(1.0 - pow(hp.beta1, (double)hp.step));
  h.bc2 = (float)(1.0 - pow(hp.beta2, (double)hp.step));
  h.lr = (float)hp.lr;
  h.eps = (float)hp.eps;
  h.lrwd = (float)(hp.lr * hp.weight_decay);
  h.lr_m = (float)(hp.lr / (1.0 - pow(hp.beta1, (double)hp.step)));
  h.root_v = (float)(1.0 / sqrt(1.0 - pow(hp.beta2, (double)hp.step)));
  // The codes of weights that are stepped in runs: the blocks' tiles read w again.
  auto blocks = [&](TileRows& l, int k, int dt) {
    uint32_t tiles = 0;
    TileRows some;
    int n = 0;
    for (int i = 0; i < k; ++i) {
      if (l.row[i].dt != dt) continue;
      some.row[n] = l.row[i];
      some.row[n++].first = tiles;
      tiles += tiles_of(l.row[i]);
    }
    if (n == 0) return (int)NOVAQ_OK;
    const void* kern = dt == E4M3 ? reinterpret_cast<const void*>(&step_blocks_kernel<E4M3>)
                                  : reinterpret_cast<const void*>(&step_blocks_kernel<E5M2>);
    void* args[] = {&some, &n};
    (void)hipLaunchKernel(kern, dim3(tiles), dim3(BQ_THREADS), args, 0, st);
    return check_launch();
  };
  // Tiles that fill the card (8 weights of 4096 x 4096, fp32 states 741 us, in runs 824;
  // 8-bit states 471 and 514; 256 tiles 23.1 and 27.4, in 8 bits 16.5 and 23.2): a few take
  // longer than both launches (64 tiles 13.8 and 11.8, 8 tiles 13.9 and 9.0).
  int64_t fitting = 0, bytes = 0, elements = 0;
  for (int64_t i = 0; i < count; ++i) {
    const novaq_adamw_tensor& t = list[i];
    if (fits_tiles(t)) fitting += ((t.rows + 127) / 128) * ((t.cols + 127) / 128);
    elements += t.n;
    bytes += t.n * (4 + (t.grad_dtype == F32 ? 4 : 2) + (t.m_exponents ? 2 : 8));
  }
  const bool in_tiles = fitting >= 256, past = bytes > (int64_t)1 << 28;
  uint32_t base = 0;
  for (int64_t at = 0; at < count;) {
    // the next rows: steps in runs, those with their blocks, and blocks that remain
    StepRows l;
    TileRows tl, bl;
    int k = 0, kt = 0, kb = 0;
    uint32_t tiles = 0;
    bool clear = false;
    const int64_t from = at;
    for (; at < count && k < STEP_ROWS && kt < TILE_ROWS && kb < TILE_ROWS; ++at) {
      const novaq_adamw_tensor& t = list[at];
      if (t.n == 0 && !t.amax_scale) continue;
      const bool s8 = t.m_exponents != nullptr;
      const bool decay = hp.weight_decay > 0.0 && t.decay;
      auto* me = static_cast<uint8_t*>(t.m_exponents);
      auto* ve = static_cast<uint8_t*>(t.v_exponents);
      const uint32_t first = base;
      base += (uint32_t)((t.n + 127) / 128 * 128);
      if (steps_alone(t, elements)) continue;
      if (t.codes && !t.amax_scale) {
        const TileRow r{t.w, t.grad, t.m, t.v, me, ve,
                        BlockOut{static_cast<uint8_t*>(t.codes), static_cast<uint8_t*>(t.exponents),
                                 static_cast<uint8_t*>(t.codes_t),
                                 static_cast<uint8_t*>(t.exponents_t)},
                        (int32_t)t.rows, (int32_t)t.cols, tiles, first, (uint8_t)t.grad_dtype, decay,
                        s8, (uint8_t)t.q_dtype};
        if (in_tiles && fits_tiles(t)) {
          tl.row[kt++] = r;
          tiles += tiles_of(r);
          continue;
        }
        bl.row[kb++] = r;
      }
      const uintptr_t ga = t.grad_dtype == F32 ? 16 : 8, sa = s8 ? 4 : 16;
      StepRow& r = l.row[k++];
      r = StepRow{};
      r.w = t.w, r.g = t.grad, r.m = t.m, r.v = t.v;
      r.me = me, r.ve = ve;
      r.amax = reinterpret_cast<uint32_t*>(t.amax_scale);
      r.n = t.n;
      r.gt = (uint8_t)t.grad_dtype;
      r.decay = decay;
      r.s8 = s8;
      r.vec = on(t.w, 16) && on(t.grad, ga) && on(t.m, sa) && on(t.v, sa);
      r.base = first;
      clear |= r.amax != nullptr;
    }
    int64_t runs = 0;
    for (int i = 0; i < k; ++i) {
      const int run = step_run_length(l.row[i].s8);
      l.row[i].first = (uint32_t)runs;
      runs += (l.row[i].n + run - 1) / run;
    }
    if (runs > 0x7FFFFFFF) return NOVAQ_ENOTSUP;
    if (clear) {
      hipLaunchKernelGGL(step_clear_kernel, dim3(1), dim3(64), 0, st, l, k);
      const int rc = check_launch();
      if (rc != NOVAQ_OK) return rc;
    }
    if (runs > 0) {
      const dim3 grid((unsigned)std::min<int64_t>(runs, 1 << 23));
      if (past)
        hipLaunchKernelGGL(step_kernel<true>, grid, dim3(256), 0, st, l, k, (uint32_t)runs, h, key);
      else
        hipLaunchKernelGGL(step_kernel<false>, grid, dim3(256), 0, st, l, k, (uint32_t)runs, h, key);
      const int rc = check_launch();
      if (rc != NOVAQ_OK) return rc;
    }
    if (kt > 0) {
      hipLaunchKernelGGL(step_tile_kernel, dim3(tiles), dim3(BQ_THREADS), 0, st, tl, kt, h, key);
      const int rc = check_launch();
      if (rc != NOVAQ_OK) return rc;
    }
    for (const int dt : {E4M3, E5M2}) {
      const int rc = blocks(bl, kb, dt);
      if (rc != NOVAQ_OK) return rc;
    }
    for (int64_t i = from; i < at; ++i) {
      const novaq_adamw_tensor& t = list[i];
      if (!t.amax_scale) continue;
      int rc = NOVAQ_OK;
      if (steps_alone(t, elements))
        rc = adamw_launch(t.w, static_cast<const float*>(t.grad), static_cast<float*>(t.m),
                          static_cast<float*>(t.v), t.n, hp.lr, hp.beta1, hp.beta2, hp.eps,
                          hp.weight_decay, hp.step, t.decay, t.amax_scale, st);
      if (rc == NOVAQ_OK)
        rc = cast_launch(t.w, F32, t.codes, t.q_dtype, t.n, 2, t.amax_scale, t.amax_scale + 1, st);
      if (rc != NOVAQ_OK) return rc;
    }
  }
  return NOVAQ_OK;
}

int state_decode_launch(const void* m, const void* me, const void* v, const void* ve, int64_t n,
                        void* om, void* ov, int out_dtype, hipStream_t st) {
  const bool vec = on(m, 4) && on(v, 4);
  // (8 elements a lane and no more, the values past the caches: 336 M elements 405 us in
  // 16384 workgroups, 343 so, 326 with both)
  const dim3 grid((unsigned)std::min<int64_t>((n + 2047) / 2048, 1 << 22));
  auto go = [&](auto ot_) {
    hipLaunchKernelGGL((state_decode_kernel<decltype(ot_)::value>), grid, dim3(256), 0, st,
                       static_cast<const uint8_t*>(m), static_cast<const uint8_t*>(me),
                       static_cast<const uint8_t*>(v), static_cast<const uint8_t*>(ve), n, om, ov,
                       vec);
    return check_launch();
  };
  switch (out_dtype) {
    case F32: return go(std::integral_constant<int, F32>{});
    case F16: return go(std::integral_constant<int, F16>{});
    default: return go(std::integral_constant<int, BF16>{});
  }
}

}  // namespace novaq
