// Softmax cross entropy of a linear head over a large vocabulary, and its
// gradients, without keeping the logits.  With x (N, D), a table W (V, D) of
// codes and its scale s:
//
//   l[n, v]  = s * sum_d x[n, d] dec(W[v, d])
//   lse[n]   = log sum_v exp(l[n, v])
//   loss[n]  = lse[n] - l[n, t[n]]             (0 where t[n] is ignore_index)
//   P[n, v]  = f[n] (exp(l[n, v] - lse[n]) - [v = t[n]])
//   grad_x   = g s P dec(W),  grad_W = g P^T x
//
// f[n] is 0 for ignored rows and else 1 (reduction mean: g = upstream / count,
// sum: g = upstream).  With a gradient for each row (u[n]; row_factors) P takes its
// digits and at most 12 of its binary places, grad_x's rows the power of two that
// is left when they are stored, and grad_W's product a copy of x with the rest of
// it: rows of very different gradients, infinite ones and NaN among them, leave
// one another's grad_x alone.
//
// The vocabulary is walked in pieces.  The forward multiplies a piece's rows
// with x and reduces each tile of logits to one (maximum, sum of 2^(l2 -
// maximum)) a row, l2 = l log2(e); a last kernel joins a row's tiles.  The
// backward computes a piece's logits again, stores P of that piece in 16 bits
// and multiplies it with the piece (grad_x, summed over the pieces in fp32)
// and with x (grad_W's rows of the piece): 8 N V D operations for both, 6 of
// them needed by any method.  Where the logits are so few that their tiles leave
// CUs idle, the products' K is split and the fp32 parts stored (loss_logits_kernel).
//
// Types: the products run in 16 bits, f16 where x is f16 and bf16 otherwise;
// FP8 and FP4 codes are exact in both, fp32 x or W and 16-bit W of the other
// type are rounded to nearest even.  P is rounded to the same type before its
// products (half an ulp of 2^-8 or 2^-11: the size of the gradients' own
// rounding where they are stored in 16 bits); in f16 it carries a factor of
// 2^14, which keeps probabilities down to 2^-28 in its normal range (2^-16 in a row
// whose own gradient is 2^-23 of the largest or less).  Logits,
// maxima, sums, lse and all accumulation are fp32; the loss over the rows is
// summed in fp64.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "novaq_internal.h"
#include "token_gemm.h"
#include "token_io.h"
#include "token_stream.h"

namespace novaq {
namespace {

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;
constexpr int T_NONE = -1, T_BAD = -2;  // no loss; an id outside the vocabulary

// The row pitch of P and of the 16-bit copies: their width and 128 elements more,
// so that rows of a power of two do not fall on the same memory channels
// (grad_x's product of 4096 x 4096 x 8192 reads 256 rows of P at a time: 367 us
// without, 279 with).
constexpr int64_t row_pitch(int64_t width) { return width + 128; }

size_t align256(size_t b) { return (b + 255) & ~(size_t)255; }

// A 16-bit copy: dst (rows x dp, pitch elements apart, dp % 64 == 0) = src (rows x
// D, stored as st) in the products' type, zeros past D and in the rows whose id is
// `ignore` (ids may be null).
struct CopyJob {
  const uint8_t* src;
  uint16_t* dst;
  int64_t rows, D, dp, pitch;
  int st;
  const void* ids;
  int bits;
  int64_t ignore;
  FastDiv by_per;  // of dp / 8
};

template <int CT, int ST, bool VEC>
__device__ __forceinline__ void copy_rows(const CopyJob& j, int64_t first, int64_t step) {
  constexpr int A = 4;  // units of 8 elements loaded before the first is stored
  const uint32_t per = (uint32_t)(j.dp / 8);
  const int64_t total = j.rows * per, rb = row_bytes(ST, j.D);
  for (int64_t q0 = first; q0 < total; q0 += A * step) {
    // codes stay codes until they are stored: two a convert
    constexpr bool codes = VEC && (ST == E4M3 || ST == E5M2 || ST == E2M1);
    float v[A][8];
    ti_u32x2 code[A];
    uint16_t* to[A];
#pragma unroll
    for (int x = 0; x < A; ++x) {
      const int64_t q = min(q0 + x * step, total - 1);
      const int64_t row = total < ((int64_t)1 << 31) ? (int64_t)fdiv((uint32_t)q, j.by_per)
                                                     : q / per;
      const int64_t c = (q - row * per) * 8;
      to[x] = j.dst + row * j.pitch + c;
      const bool here = c < j.D && !(j.ids && token_at(j.ids, j.bits, row) == j.ignore);
      if constexpr (codes) {
        code[x] = ti_u32x2{0, 0};
        const uint8_t* p = j.src + row * rb + (ST == E2M1 ? c / 2 : c);
        if (here) {
          if constexpr (ST == E2M1) code[x][0] = vload<true>(reinterpret_cast<const uint32_t*>(p));
          else code[x] = vload<true>(reinterpret_cast<const ti_u32x2*>(p));
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[x][i] = 0.0f;
        if (here) load8<ST, VEC, true>(j.src + row * rb, c, j.D, v[x]);
      }
    }
#pragma unroll
    for (int x = 0; x < A; ++x) {
      if (q0 + x * step >= total) break;
      ti_u32x4 o;
      if constexpr (codes) {
        o = ts_decode8<CT, ST>(code[x][0], code[x][1]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = tg_pack2<CT>(v[x][2 * i], v[x][2 * i + 1]);
      }
      *reinterpret_cast<ti_u32x4*>(to[x]) = o;
    }
  }
}

template <int CT>
__device__ __forceinline__ void copy_job(const CopyJob& j, int64_t first, int64_t step) {
  const bool vec = j.D % 8 == 0;
  switch (j.st) {
#define NOVAQ_COPY(ST)                                     \
  case ST:                                                 \
    if (vec) copy_rows<CT, ST, true>(j, first, step);      \
    else copy_rows<CT, ST, false>(j, first, step);         \
    break;
    NOVAQ_COPY(F32)
    NOVAQ_COPY(F16)
    NOVAQ_COPY(BF16)
    NOVAQ_COPY(E4M3)
    NOVAQ_COPY(E5M2)
    NOVAQ_COPY(E2M1)
#undef NOVAQ_COPY
  }
}

// The tokens' fragments of the kernel for few rows (token_stream.h): 16 bytes a
// thread, fragment ((stage 4 + c) U + u) nt + j of 64 lanes; x (N x D) as st,
// zeros past N and D.
struct FragmentJob {
  const uint8_t* x;
  uint16_t* dst;
  int64_t N, D, total;
  int st, E, nt;
};

template <int CT, int ST, bool VEC>
__device__ __forceinline__ void fragments(const FragmentJob& f, int64_t first, int64_t step) {
  const int us = 31 - __clz(f.E / 8), ns = 31 - __clz(f.nt);  // (both powers of two)
  const int64_t rb = row_bytes(ST, f.D);
  for (int64_t q = first; q < f.total; q += step) {
    const int lane = (int)(q & 63);
    const int64_t fr = q >> 6, at = fr >> ns, pair = at >> us;  // of chunks
    const int j = (int)(fr & (f.nt - 1)), u = (int)at & (f.E / 8 - 1);
    const int64_t n = j * 32 + (lane & 31), k = f.E * (2 * pair + (lane >> 5)) + 8 * u;
    float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (n < f.N && k < f.D) load8<ST, VEC>(f.x + n * rb, k, f.D, v);
    ti_u32x4 o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = tg_pack2<CT>(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<ti_u32x4*>(f.dst + q * 8) = o;
  }
}

// Per-row state: targets as int32 (T_NONE, T_BAD), the row factors f (NaN for
// T_BAD, so its gradients show; may be null), scal[0] = g, scal[1] = the number
// of rows with a loss.
// grad: one value, or one a row (per_row; then fx and fw too), or null (1).
struct RowsJob {
  const void* ids;
  int bits;
  int64_t ignore, N, V;
  const float* grad;
  int per_row, mean;
  int* targets;
  float* f;
  float* scal;
  float *fx, *fw;  // what grad_x's rows are scaled by, and x's for grad_W
};

// The exponent e of a finite a > 0: 2^e <= a < 2^(e + 1).
__device__ __forceinline__ int exponent(float a) {
  const int e = (int)(f2u(a) >> 23);
  return e > 0 ? e - 127 : 31 - __clz(f2u(a)) - 149;
}

// The gradient u of one row as f fx = u and f fw 2^top = u, 2^top being the power of
// two in the largest finite one.  With d the places that u lies below that: f is u's
// digits (1 <= |f| < 2) moved down by half of d, but 12 places at most, fw = 2^-(the
// other places), both exact.  So P in f16 (a factor of 2^14 above one) holds
// probabilities down to 2^-16 in its normal range however small a row's gradient is,
// and x fw loses bits only where it falls under 2^-14.  An infinite or NaN u is kept
// out of P, which both products read.
__device__ __forceinline__ void row_factors(float u, int top, float& f, float& fx, float& fw) {
  const float a = fabsf(u);
  if (!(a < INFINITY)) {
    f = 1.0f, fx = fw = u;
  } else if (a == 0.0f) {
    f = 0.0f, fx = fw = 1.0f;
  } else {
    const int e = exponent(a), d = top - e, down = min(d - d / 2, 12);
    f = ldexpf(u, -e - down);
    fx = ldexpf(1.0f, e + down);
    fw = ldexpf(1.0f, down - d);
  }
}

__device__ __forceinline__ void rows_job(const RowsJob& r, int* cnt, float* top) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int c = 0;
  float m = 0.0f;
  for (int64_t n0 = tid; n0 < r.N; n0 += 2048) {
    int64_t t[8];
#pragma unroll
    for (int x = 0; x < 8; ++x) t[x] = token_at(r.ids, r.bits, min(n0 + 256 * x, r.N - 1));
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      const int64_t n = n0 + 256 * x;
      if (n >= r.N) continue;
      const int k = t[x] == r.ignore ? T_NONE : t[x] < 0 || t[x] >= r.V ? T_BAD : (int)t[x];
      r.targets[n] = k;
      c += k != T_NONE;
      if (r.per_row && k != T_NONE && fabsf(r.grad[n]) < INFINITY) m = fmaxf(m, fabsf(r.grad[n]));
      if (r.f && !r.per_row) r.f[n] = k == T_NONE ? 0.0f : k == T_BAD ? u2f(0x7FC00000u) : 1.0f;
    }
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    c += __shfl_xor(c, d);
    m = fmaxf(m, __shfl_xor(m, d));
  }
  if (lane == 0) cnt[wave] = c, top[wave] = m;
  __syncthreads();
  c = 0, m = 0.0f;
#pragma unroll
  for (int w = 0; w < 4; ++w) c += cnt[w], m = fmaxf(m, top[w]);
  const int e = m > 0.0f ? exponent(m) : 0;
  if (tid == 0) {
    float g = r.per_row ? ldexpf(1.0f, e) : r.grad ? *r.grad : 1.0f;
    if (r.mean) g = c > 0 ? g / (float)c : 0.0f;
    r.scal[0] = g;
    r.scal[1] = (float)c;
  }
  if (r.f && r.per_row)
    for (int64_t n = tid; n < r.N; n += 256) {
      const int k = r.targets[n];
      float f = k == T_NONE ? 0.0f : u2f(0x7FC00000u), fx = 1.0f, fw = 1.0f;
      if (k >= 0) row_factors(r.grad[n], e, f, fx, fw);
      r.f[n] = f, r.fx[n] = fx, r.fw[n] = fw;
    }
}

// What a call needs before its products, in one launch: workgroup 0 the rows, the
// next ones x's copy (or fragments), the rest the table's first piece; and for the
// later pieces their copies alone (rows.N, x.rows and frag.total 0).
template <int CT>
__global__ __launch_bounds__(256) void loss_prep_kernel(RowsJob rows, CopyJob x, FragmentJob frag,
                                                         CopyJob w, int xblocks) {
  __shared__ int cnt[4];
  __shared__ float top[4];
  int b = blockIdx.x;
  if (rows.N > 0) {
    if (b == 0) {
      rows_job(rows, cnt, top);
      return;
    }
    --b;
  }
  if (b < xblocks) {
    const int64_t first = (int64_t)b * 256 + threadIdx.x, step = (int64_t)xblocks * 256;
    if (x.rows > 0) copy_job<CT>(x, first, step);
    else if (frag.st == F32) {
      if (frag.D % 8 == 0) fragments<CT, F32, true>(frag, first, step);
      else fragments<CT, F32, false>(frag, first, step);
    } else {  // (f16 and bf16 x are in the products' type)
      if (frag.D % 8 == 0) fragments<CT, CT, true>(frag, first, step);
      else fragments<CT, CT, false>(frag, first, step);
    }
    return;
  }
  b -= xblocks;
  const int wblocks = gridDim.x - xblocks - (rows.N > 0);
  copy_job<CT>(w, (int64_t)b * 256 + threadIdx.x, (int64_t)wblocks * 256);
}

template <int CT>
int prep_launch(const RowsJob& rows, CopyJob x, const FragmentJob& frag, CopyJob w,
                hipStream_t stream) {
  auto blocks = [](int64_t units) { return (int)std::min<int64_t>((units + 1023) / 1024, 16384); };
  if (x.rows > 0) x.by_per = fast_div((uint32_t)(x.dp / 8));
  if (w.rows > 0) w.by_per = fast_div((uint32_t)(w.dp / 8));
  // (four units a thread; of the few fragments one, which are waited for)
  const int xb = x.rows > 0 ? blocks(x.rows * (x.dp / 8)) : blocks(frag.total * 4);
  const int wb = blocks(w.rows * (w.dp / 8));
  const int all = (rows.N > 0) + xb + wb;
  if (all == 0) return NOVAQ_OK;
  hipLaunchKernelGGL(loss_prep_kernel<CT>, dim3(all), dim3(256), 0, stream, rows, x, frag, w, xb);
  return check_launch();
}

// x's rows times fw, for grad_W's product where each row has a gradient of its own:
// N x dp 16-bit values (pitch elements apart), 8 a thread.
template <int CT>
__global__ __launch_bounds__(256) void loss_scaled_x_kernel(const uint16_t* __restrict__ x,
                                                            const float* __restrict__ fw, int64_t N,
                                                            int64_t dp, int64_t pitch,
                                                            uint16_t* __restrict__ out) {
  const int64_t per = dp / 8, total = N * per;
  for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < total; q += (int64_t)gridDim.x * 256) {
    const int64_t n = q / per, at = n * pitch + (q - n * per) * 8;
    const float a = fw[n];
    float v[8];
    load8<CT, true>(reinterpret_cast<const uint8_t*>(x), at, 0, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= a;
    tg_u32x4 o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = tg_pack2<CT>(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<tg_u32x4*>(out + at) = o;
  }
}

// 8 workgroups in a row go to the 8 XCDs: those of one XCD take a compact
// group of tiles, 4 along M.
__device__ __forceinline__ void tile_of(int t, int tm, int tn, int& m, int& n) {
  const int T = tm * tn;
  if ((T & 7) == 0) t = (t & 7) * (T >> 3) + (t >> 3);
  constexpr int GM = 4;
  const int group = t / (GM * tn), first = group * GM, gm = min(tm - first, GM);
  const int rem = t - group * GM * tn;
  m = first + rem % gm;
  n = rem / gm;
}

// log2(e) times the scale; 0 (all logits 0) becomes the smallest normal number,
// which leaves them 0 and a product with an infinity infinite.
__device__ __forceinline__ float logit_factor(const float* w_scale) {
  const float c2 = (w_scale ? *w_scale : 1.0f) * LOG2E;
  return c2 == 0.0f ? 0x1p-126f : c2;
}

// (maximum, sum of 2^(l2 - maximum)) of two disjoint sets of one token's logits.
__device__ __forceinline__ float2 join_stats(const float2& a, const float2& b) {
  const float m = fmaxf(a.x, b.x), z = m == -INFINITY ? 0.0f : m;
  return float2{m, a.y * __builtin_amdgcn_exp2f(a.x - z) + b.y * __builtin_amdgcn_exp2f(b.x - z)};
}

// The statistics of the I x R products of one token that a lane holds.  at(i, r)
// is the product of row row(i, r) (from the lane's own first row); those from
// `rows` on do not exist.  mine: the row of the token's target, or -1; its logit
// goes to *tlogit.
template <int I, int R, class F, class G>
__device__ __forceinline__ float2 column_stats(F&& at, G&& row, bool ragged, int rows, int mine,
                                               float c2, float* tlogit) {
  if (__ballot(mine >= 0)) {  // (few tiles hold a target of their tokens)
    float l = 0.0f;
    bool here = false;
#pragma unroll
    for (int i = 0; i < I; ++i)
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const bool hit = row(i, r) == mine;
        l = hit ? at(i, r) : l;
        here |= hit;
      }
    if (here) *tlogit = l * c2;
  }
  if (ragged) {  // below every logit, in either sign of the scale
#pragma unroll
    for (int i = 0; i < I; ++i)
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (row(i, r) >= rows) at(i, r) = c2 < 0.0f ? INFINITY : -INFINITY;
  }
  float top = at(0, 0);
  if (c2 < 0.0f) {
#pragma unroll
    for (int i = 0; i < I; ++i)
#pragma unroll
      for (int r = 0; r < R; ++r) top = fminf(top, at(i, r));
  } else {
#pragma unroll
    for (int i = 0; i < I; ++i)
#pragma unroll
      for (int r = 0; r < R; ++r) top = fmaxf(top, at(i, r));
  }
  const float m = top * c2, z = m == -INFINITY ? 0.0f : m;
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < I; ++i)
#pragma unroll
    for (int r = 0; r < R; ++r) s += __builtin_amdgcn_exp2f(fmaf(at(i, r), c2, -z));
  return float2{m, s};
}

// The same of the lanes `d` apart, joined.
__device__ __forceinline__ float2 across(const float2& a, int d) {
  return join_stats(a, float2{__shfl_xor(a.x, d), __shfl_xor(a.y, d)});
}

// The row of token n's target among the `many` rows from r0 on, or -1.
__device__ __forceinline__ int target_row(int t, int64_t r0, int many) {
  const int64_t d = (int64_t)t - r0;
  return t < 0 || d < 0 || d >= many ? -1 : (int)d;
}

// The forward's tile: BM vocabulary rows (from v0 + m0) x BN tokens.  A lane
// holds one token's logits of a column, so a row's maximum and sum stay in
// registers but for the exchange between the four lanes and the two waves that
// share the tokens.  4096 x 4096 x 131072: 3.27 ms = 1.35 PFLOP/s, the matrix cores'
// rate at the clock that the card's power allows (a library product of that size:
// 1.31 to 1.45).
template <int CT, class G>
__global__ __launch_bounds__(G::NTH, 1) void loss_stats_kernel(
    TokenOp w, TokenOp x, int64_t dp, const float* __restrict__ w_scale, int64_t v0, int64_t N,
    const int* __restrict__ targets, float2* __restrict__ stats, int64_t vtiles,
    float* __restrict__ tlogit, int tm, int tn) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  int mi, ni;
  tile_of(blockIdx.x, tm, tn, mi, ni);
  const int64_t m0 = (int64_t)mi * G::BM, n0 = (int64_t)ni * G::BN;
  typename G::Acc acc;
  G::run(acc, w, x, m0, n0, dp, 0, (int)(dp / 64), lds);

  const float c2 = logit_factor(w_scale);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4, c = lane & 15;
  const int wm = (wave % G::WGM) * G::WM, wn = (wave / G::WGM) * G::WN;
  const int rows = (int)min((int64_t)G::BM, w.rows - m0) - wm - 4 * q;  // of this lane
  const bool ragged = w.rows - m0 < G::BM;
  float2* part = reinterpret_cast<float2*>(lds);  // [BN]
  float2 st[G::NT];
#pragma unroll
  for (int j = 0; j < G::NT; ++j) {
    const int64_t n = n0 + wn + 16 * j + c;
    const int t = n < N ? targets[n] : T_NONE;
    st[j] = column_stats<G::MT, 4>([&](int i, int r) -> float& { return ((float*)&acc[i][j])[r]; },
                                   [](int i, int r) { return 16 * i + r; }, ragged, rows,
                                   target_row(t, v0 + m0 + wm + 4 * q, G::WM), c2, tlogit + n);
    st[j] = across(across(st[j], 16), 32);
    if ((wave & 1) && q == 0) part[wn + 16 * j + c] = st[j];
    __builtin_amdgcn_sched_barrier(0);  // (a column's values at a time in registers)
  }
  __syncthreads();
  if ((wave & 1) == 0 && q == 0) {
#pragma unroll
    for (int j = 0; j < G::NT; ++j) {
      const int64_t n = n0 + wn + 16 * j + c;
      const float2 o = join_stats(st[j], part[wn + 16 * j + c]);
      if (n < N) stats[n * vtiles + (v0 + m0) / G::BM] = o;
    }
  }
}

// The same for at most 128 tokens, the table read as stored.
template <int CT, int WT, class S>
__global__ __launch_bounds__(S::NTH, 1) void loss_stream_kernel(
    const uint8_t* __restrict__ w, int64_t V, int64_t rb, const uint8_t* __restrict__ xf,
    int stages, const float* __restrict__ w_scale, int64_t N, const int* __restrict__ targets,
    float2* __restrict__ stats, int64_t vtiles, float* __restrict__ tlogit) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int64_t r0 = (int64_t)blockIdx.x * S::ROWS;
  typename S::Acc acc;
  // (8 workgroups in a row are on 8 XCDs)
  S::run(acc, w, V, rb, r0, xf, stages, (int)((blockIdx.x >> 3) % (unsigned)stages), lds);

  const float c2 = logit_factor(w_scale);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
  const int rows = (int)min((int64_t)S::ROWS, V - r0) - 32 * wave - 4 * half;
  const bool ragged = V - r0 < S::ROWS;
  float2* part = reinterpret_cast<float2*>(lds);  // [waves][tokens]
#pragma unroll
  for (int j = 0; j < S::NT; ++j) {
    const int64_t n = 32 * j + (lane & 31);
    const int t = n < N ? targets[n] : T_NONE;
    const float2 st = across(
        column_stats<1, 16>([&](int, int r) -> float& { return ((float*)&acc[j])[r]; },
                            [](int, int r) { return 8 * (r >> 2) + (r & 3); }, ragged, rows,
                            target_row(t, r0 + 32 * wave + 4 * half, 32), c2, tlogit + n),
        32);
    if (half == 0) part[wave * 32 * S::NT + 32 * j + (lane & 31)] = st;
  }
  __syncthreads();
  if ((int)threadIdx.x < 32 * S::NT && (int64_t)threadIdx.x < N) {
    float2 o = part[threadIdx.x];
    for (int v = 1; v < S::NTH / 64; ++v) o = join_stats(o, part[v * 32 * S::NT + threadIdx.x]);
    stats[(int64_t)threadIdx.x * vtiles + blockIdx.x] = o;
  }
}

// The rows' losses summed in fp64 in a fixed order by 16 waves, over the count for
// mean (0 where no row has a loss).
__device__ __forceinline__ void sum_losses(const float* each, int64_t N, int mean,
                                           const float* scal, float* out, double* part) {
  double s = 0.0;
#pragma unroll 4
  for (int64_t n = threadIdx.x; n < N; n += 1024) s += (double)each[n];
#pragma unroll
  for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0.0;
    for (int w = 0; w < 16; ++w) s += part[w];
    if (mean) s = scal[1] > 0.0f ? s / (double)scal[1] : 0.0;
    *out = (float)s;
  }
}

__global__ __launch_bounds__(1024) void loss_sum_kernel(const float* __restrict__ each, int64_t N,
                                                        int mean, const float* __restrict__ scal,
                                                        float* __restrict__ out) {
  __shared__ double part[16];
  sum_losses(each, N, mean, scal, out, part);
}

// One wave a row joins the tiles' (maximum, sum) pairs: lse and the loss.  A
// single workgroup (grid 1) takes all rows and sums their losses into `out`.
__global__ __launch_bounds__(1024) void loss_join_kernel(const float2* __restrict__ stats,
                                                         int64_t vtiles, int64_t N,
                                                         const int* __restrict__ targets,
                                                         const float* __restrict__ tlogit,
                                                         float* __restrict__ lse, float* loss,
                                                         int mean, const float* __restrict__ scal,
                                                         float* __restrict__ out) {
  __shared__ double part[16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int64_t n = (int64_t)blockIdx.x * 16 + wave; n < N; n += (int64_t)gridDim.x * 16) {
    float2 a = {-INFINITY, 0.0f};
#pragma unroll 4
    for (int64_t i = lane; i < vtiles; i += 64) a = join_stats(a, stats[n * vtiles + i]);
#pragma unroll
    for (int d = 32; d; d >>= 1) a = join_stats(a, float2{__shfl_xor(a.x, d), __shfl_xor(a.y, d)});
    if (lane == 0) {
      const float l2 = a.x + log2f(a.y);
      const int t = targets[n];
      lse[n] = l2 * LN2;
      // (the difference in base 2: the factor's rounding falls on the loss alone)
      loss[n] = t == T_NONE ? 0.0f : t == T_BAD ? u2f(0x7FC00000u) : (l2 - tlogit[n]) * LN2;
    }
  }
  if (gridDim.x > 1 || !out) return;
  __syncthreads();
  sum_losses(loss, N, mean, scal, out, part);
}

// The backward's P of one piece: the forward's tile, then f (2^(l2 - lse2) -
// [v = t]) in 16 bits at P[n][v] (pitch vp; the piece's columns past the
// vocabulary are zeros), through LDS so that rows leave in whole lines.  A piece of
// 16384 classes at 4096 x 4096: 426 us = 1.29 PFLOP/s.
template <int CT, class G>
__global__ __launch_bounds__(G::NTH, 1) void loss_prob_kernel(
    TokenOp w, TokenOp x, int64_t dp, const float* __restrict__ w_scale, int64_t v0, int64_t N,
    const int* __restrict__ targets, const float* __restrict__ f, const float* __restrict__ lse,
    float pscale, uint16_t* __restrict__ P, int64_t vp, int tm, int tn) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  int mi, ni;
  tile_of(blockIdx.x, tm, tn, mi, ni);
  const int64_t m0 = (int64_t)mi * G::BM, n0 = (int64_t)ni * G::BN;
  typename G::Acc acc;
  G::run(acc, w, x, m0, n0, dp, 0, (int)(dp / 64), lds);

  const float c2 = logit_factor(w_scale);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4;
  const int wm = (wave % G::WGM) * G::WM, wn = (wave / G::WGM) * G::WN;
  const int rows = (int)max((int64_t)0, min((int64_t)G::BM, w.rows - m0)) - wm - 4 * q;
  const bool ragged = w.rows - m0 < G::BM;
  // token rows of BM 16-bit values and 16 bytes more, so that the rows that a
  // store touches start in different banks
  constexpr int PITCH = G::BM * 2 + 16;
#pragma unroll
  for (int j = 0; j < G::NT; ++j) {
    const int col = wn + 16 * j + (lane & 15);
    const int64_t n = n0 + col;
    const bool in = n < N;
    const int t = in ? targets[n] : T_NONE;
    const int mine = target_row(t, v0 + m0 + wm + 4 * q, G::WM);
    // (an ignored row's x is zeros and its f 0: with any finite lse P is 0)
    const float fn = in ? f[n] * pscale : 0.0f;
    const float l2 = in && t != T_NONE ? lse[n] * LOG2E : 0.0f;
    uint8_t* row = lds + col * PITCH + (wm + 4 * q) * 2;
#pragma unroll
    for (int i = 0; i < G::MT; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        acc[i][j][r] = __builtin_amdgcn_exp2f(fmaf(acc[i][j][r], c2, -l2));
    if (__ballot(mine >= 0)) {  // (few tiles hold a target of their tokens)
#pragma unroll
      for (int i = 0; i < G::MT; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (16 * i + r == mine) acc[i][j][r] -= 1.0f;
    }
    if (ragged) {
#pragma unroll
      for (int i = 0; i < G::MT; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (16 * i + r >= rows) acc[i][j][r] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < G::MT; ++i)
      *reinterpret_cast<tg_u32x2*>(row + 32 * i) =
          tg_u32x2{tg_pack2<CT>(acc[i][j][0] * fn, acc[i][j][1] * fn),
                   tg_pack2<CT>(acc[i][j][2] * fn, acc[i][j][3] * fn)};
  }
  __syncthreads();
  constexpr int CPR = G::BM / 8;  // 16-byte chunks a token row
  for (int q = threadIdx.x; q < G::BN * CPR; q += G::NTH) {
    const int r = q / CPR, c = q % CPR;
    if (n0 + r < N)
      *reinterpret_cast<tg_u32x4*>(P + (n0 + r) * vp + m0 + c * 8) =
          *reinterpret_cast<const tg_u32x4*>(lds + r * PITCH + c * 16);
  }
}

// --------------------------------------------------------------------------
// few tiles of logits: their K split over the CUs

// This split's fp32 products of one tile, at sums[split][n][v] (pitch vp).
template <int CT, class G>
__global__ __launch_bounds__(G::NTH, 1) void loss_logits_kernel(TokenOp w, TokenOp x, int64_t dp,
                                                                int64_t N, int splits,
                                                                float* __restrict__ sums,
                                                                int64_t vp, int tm, int tn) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  int mi, ni;
  const int split = blockIdx.x / (tm * tn), blocks = (int)(dp / 64);
  tile_of(blockIdx.x % (tm * tn), tm, tn, mi, ni);
  const int64_t m0 = (int64_t)mi * G::BM, n0 = (int64_t)ni * G::BN;
  typename G::Acc acc;
  G::run(acc, w, x, m0, n0, dp, blocks * split / splits, blocks * (split + 1) / splits, lds);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4;
  const int wm = (wave % G::WGM) * G::WM, wn = (wave / G::WGM) * G::WN;
#pragma unroll
  for (int j = 0; j < G::NT; ++j) {
    const int64_t n = n0 + wn + 16 * j + (lane & 15);
    float* p = sums + ((int64_t)split * N + n) * vp + m0 + wm + 4 * q;
    if (n < N) {
#pragma unroll
      for (int i = 0; i < G::MT; ++i) *reinterpret_cast<tg_f32x4*>(p + 16 * i) = acc[i][j];
    }
  }
}

// Four products of token n from v on, their splits added in order.
__device__ __forceinline__ tg_f32x4 split_sum(const float* sums, int splits, int64_t N, int64_t vp,
                                              int64_t n, int64_t v) {
  tg_f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
  for (int k = 0; k < splits; ++k) {
    const tg_f32x4 o = *reinterpret_cast<const tg_f32x4*>(sums + ((int64_t)k * N + n) * vp + v);
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] += o[i];
  }
  return s;
}

// A token's lse and loss from its split logits, one workgroup.
__global__ __launch_bounds__(256) void loss_rows_kernel(const float* __restrict__ sums, int splits,
                                                        int64_t N, int64_t V, int64_t vp,
                                                        const float* __restrict__ w_scale,
                                                        const int* __restrict__ targets,
                                                        float* __restrict__ lse, float* loss) {
  __shared__ float2 part[4];
  __shared__ float tlogit;
  const int64_t n = blockIdx.x;
  const int t = targets[n];
  const float c2 = logit_factor(w_scale);
  float2 a = {-INFINITY, 0.0f};
  for (int64_t v = threadIdx.x * 4; v < V; v += 1024) {
    const tg_f32x4 s = split_sum(sums, splits, N, vp, n, v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (v + i >= V) continue;
      a = join_stats(a, float2{s[i] * c2, 1.0f});
      if (v + i == t) tlogit = s[i] * c2;
    }
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) a = across(a, d);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = a;
  __syncthreads();
  if (threadIdx.x > 0) return;
  for (int w = 1; w < 4; ++w) a = join_stats(a, part[w]);
  const float l2 = a.x + log2f(a.y);
  lse[n] = l2 * LN2;
  loss[n] = t == T_NONE ? 0.0f : t == T_BAD ? u2f(0x7FC00000u) : (l2 - tlogit) * LN2;
}

// The backward's P (as in loss_prob_kernel) of a piece from its split logits: 8
// classes a thread, a token a grid row.
template <int CT>
__global__ __launch_bounds__(256) void loss_prob_rows_kernel(
    const float* __restrict__ sums, int splits, int64_t N, int64_t vc, int64_t vp, int64_t v0,
    const float* __restrict__ w_scale, const int* __restrict__ targets,
    const float* __restrict__ f, const float* __restrict__ lse, float pscale,
    uint16_t* __restrict__ P, int64_t pitch) {
  const int64_t n = blockIdx.y, v = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
  if (v >= vp) return;
  const int t = targets[n];
  const float c2 = logit_factor(w_scale), fn = f[n] * pscale;
  const float l2 = t != T_NONE ? lse[n] * LOG2E : 0.0f;
  tg_u32x4 o = {0, 0, 0, 0};
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (v + 4 * h >= vc) break;
    tg_f32x4 s = split_sum(sums, splits, N, vp, n, v + 4 * h);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t at = v + 4 * h + i;
      const float e = __builtin_amdgcn_exp2f(fmaf(s[i], c2, -l2)) - (v0 + at == t ? 1.0f : 0.0f);
      s[i] = at < vc ? e * fn : 0.0f;
    }
    o[2 * h] = tg_pack2<CT>(s[0], s[1]);
    o[2 * h + 1] = tg_pack2<CT>(s[2], s[3]);
  }
  *reinterpret_cast<tg_u32x4*>(P + n * pitch + v) = o;
}

// The gradients' products of one piece.
struct GradsJob {
  TokenOp p, pt;        // P: N rows of K; and as K-strided rows of the vocabulary
  TokenOp w, x;         // the piece and x, both K-strided
  int64_t N, D, vc;     // vc: the piece's rows
  int vblocks, nblocks; // K blocks of the two products
  int splits, first;    // of grad_x's K; the first piece stores, the others add
  float* sums;          // grad_x's fp32 sums, split by split, pitch dp
  int64_t dp;
  const float* scal;
  float inv_pscale;
  uint8_t* gw;
  float* wsums;            // where grad_W's K is split: fp32 sums as above, of the piece
  int wsplits;
  int xtm, xtn, wtm, wtn;  // tiles; wtm 0: no grad_W
};

// grad_x's share of one piece: P (N x vc) times the piece's rows (vc x D), K
// blocks of this split, added to (or, first, stored in) the split's fp32 sums.
template <int CT, class G>
__device__ __forceinline__ void dx_tile(const GradsJob& g, int b, uint8_t* lds) {
  int mi, ni;
  const int split = b / (g.xtm * g.xtn);
  tile_of(b % (g.xtm * g.xtn), g.xtm, g.xtn, mi, ni);
  const int64_t m0 = (int64_t)mi * G::BM, n0 = (int64_t)ni * G::BN, N = g.N, D = g.D, dp = g.dp;
  float* sums = g.sums;
  const int first = g.first;
  typename G::Acc acc;
  G::run(acc, g.p, g.w, m0, n0, g.vc, (int)((int64_t)g.vblocks * split / g.splits),
         (int)((int64_t)g.vblocks * (split + 1) / g.splits), lds);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4;
  const int wm = (wave % G::WGM) * G::WM, wn = (wave / G::WGM) * G::WN;
  // what lies past N or D is left out by the descriptor (offsets past it)
  const int rows = (int)min((int64_t)G::BM, N - m0);
  const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
      sums + ((int64_t)split * N + m0) * dp, (short)0, rows * (int)dp * 4, 0x00020000);
  const uint32_t pitch = (uint32_t)dp * 4;
#pragma unroll
  for (int j = 0; j < G::NT; ++j) {
    const int64_t d = n0 + wn + 16 * j + (lane & 15);
    const uint32_t at = d < D ? (uint32_t)(wm + 4 * q) * pitch + (uint32_t)d * 4 : 0x80000000u;
#pragma unroll
    for (int i = 0; i < G::MT; ++i) {
      float old[4];
#pragma unroll
      for (int r = 0; r < 4; ++r)
        old[r] = first ? 0.0f
                       : u2f(__builtin_amdgcn_raw_buffer_load_b32(
                             rs, at + (16 * i + r) * pitch, 0, 0));
#pragma unroll
      for (int r = 0; r < 4; ++r)
        __builtin_amdgcn_raw_buffer_store_b32(f2u(old[r] + acc[i][j][r]), rs,
                                              at + (16 * i + r) * pitch, 0,
                                              0);
      // (16 loads in flight at a time: all of a tile's would not fit the registers)
      if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);
    }
  }
}

// A product rounded to fp32 before it is converted: the compiler makes one mixed
// instruction of a multiply and a conversion to f16, and a gradient in f16 would
// then differ from the fp32 one's rounding at ties.
__device__ __forceinline__ float rounded(float y) {
  asm("" : "+v"(y));
  return y;
}

// grad_W's rows of one piece: P^T (vc x N) times x (N x D), times g / pscale, as
// OT; or (OT SUMS), where its K is split, this split's fp32 sums.
constexpr int SUMS = -1;
template <int CT, int OT, class G>
__device__ __forceinline__ void dw_tile(const GradsJob& g, int b, uint8_t* lds) {
  int mi, ni, split = 0;
  if constexpr (OT == SUMS) split = b / (g.wtm * g.wtn), b %= g.wtm * g.wtn;
  tile_of(b, g.wtm, g.wtn, mi, ni);
  const int64_t m0 = (int64_t)mi * G::BM, n0 = (int64_t)ni * G::BN, D = g.D, vc = g.vc;
  int k0 = 0, k1 = g.nblocks;
  if constexpr (OT == SUMS) {
    k0 = (int)((int64_t)g.nblocks * split / g.wsplits);
    k1 = (int)((int64_t)g.nblocks * (split + 1) / g.wsplits);
  }
  typename G::Acc acc;
  G::run(acc, g.pt, g.x, m0, n0, g.N, k0, k1, lds);
  const float a = OT == SUMS ? 1.0f : g.scal[0] * g.inv_pscale;
  uint8_t* out = g.gw;
  int64_t ld = D;
  if constexpr (OT == SUMS) out = (uint8_t*)(g.wsums + split * vc * g.dp), ld = g.dp;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4;
  const int wm = (wave % G::WGM) * G::WM, wn = (wave / G::WGM) * G::WN;
  constexpr bool F = OT == F32 || OT == SUMS;
  constexpr int OB = F ? 4 : 2;
  const int rows = (int)min((int64_t)G::BM, vc - m0);
  const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
      out + m0 * ld * OB, (short)0, rows * (int)ld * OB, 0x00020000);
  const uint32_t pitch = (uint32_t)ld * OB;
#pragma unroll
  for (int j = 0; j < G::NT; ++j) {
    const int64_t d = n0 + wn + 16 * j + (lane & 15);
    const uint32_t at = d < D ? (uint32_t)(wm + 4 * q) * pitch + (uint32_t)d * OB : 0x80000000u;
#pragma unroll
    for (int i = 0; i < G::MT; ++i) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const uint32_t o = at + (16 * i + r) * pitch;
        const float y = OT == F16 ? rounded(acc[i][j][r] * a) : acc[i][j][r] * a;
        if constexpr (F) __builtin_amdgcn_raw_buffer_store_b32(f2u(y), rs, o, 0, 0);
        else
          __builtin_amdgcn_raw_buffer_store_b16((uint16_t)tg_pack2<OT>(y, 0.0f), rs, o, 0, 0);
      }
      if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);
    }
  }
}

// Both gradients' tiles in one launch, grad_x's first: each product alone leaves
// CUs idle in its last round (8192 x 1024 x 8192: 128 tiles of 256 x 256 each).
// Bound by the matrix cores at the clock the card's power allows: 850 us = 1.29
// PFLOP/s for a piece of 16384 classes at 4096 x 4096 (MFMA busy 67%, LDS 25%).
template <int CT, int OT, class GX, class GW>
__global__ __launch_bounds__(GX::NTH, 1) void loss_grads_kernel(GradsJob g) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int nx = g.xtm * g.xtn * g.splits;
  if ((int)blockIdx.x < nx) dx_tile<CT, GX>(g, blockIdx.x, lds);
  else dw_tile<CT, OT, GW>(g, blockIdx.x - nx, lds);
}

// A gradient = its splits' sums times g s / pscale, as OT (rows of ignored targets
// 0; with fx that of each row in g's place; grad_W has neither s nor targets): four
// columns a thread, or, with SHARE, four threads (one in each wave) that take every fourth split each and add up in their
// order.
template <int OT, bool SHARE>
__global__ __launch_bounds__(256) void loss_sums_store_kernel(const float* __restrict__ sums,
                                                            int splits, int64_t N, int64_t dp,
                                                            int64_t D,
                                                            const float* __restrict__ scal,
                                                            const float* __restrict__ w_scale,
                                                            float inv_pscale,
                                                            const int* __restrict__ targets,
                                                            const float* __restrict__ fx,
                                                            void* __restrict__ out) {
  __shared__ float4 part[SHARE ? 3 * 64 : 1];
  const float scale = w_scale ? *w_scale : 1.0f, all = scal[0] * scale * inv_pscale;
  const int64_t per = dp / 4, total = N * per;
  constexpr int STEP = SHARE ? 4 : 1, UNITS = 256 / STEP;
  const int from = SHARE ? threadIdx.x >> 6 : 0, unit = SHARE ? threadIdx.x & 63 : threadIdx.x;
  const bool vec = D % 4 == 0;
  for (int64_t q0 = (int64_t)blockIdx.x * UNITS; q0 < total; q0 += (int64_t)gridDim.x * UNITS) {
    const int64_t q = min(q0 + unit, total - 1);
    const int64_t n = q / per, c = (q - n * per) * 4;
    float v[4] = {0, 0, 0, 0};
    const float* p = sums + n * dp + c;
#pragma unroll 8
    for (int s = from; s < splits; s += STEP) {
      const float4 o = *reinterpret_cast<const float4*>(p + (int64_t)s * N * dp);
      v[0] += o.x, v[1] += o.y, v[2] += o.z, v[3] += o.w;
    }
    if constexpr (SHARE) {
      if (from > 0) part[(from - 1) * 64 + unit] = float4{v[0], v[1], v[2], v[3]};
      __syncthreads();
      if (from == 0)
        for (int w = 0; w < 3; ++w) {
          const float4 o = part[w * 64 + unit];
          v[0] += o.x, v[1] += o.y, v[2] += o.z, v[3] += o.w;
        }
      __syncthreads();
    }
    if (from > 0 || q0 + unit >= total || c >= D) continue;
    const bool none = targets && targets[n] == T_NONE;
    const float a = fx ? fx[n] * scale * inv_pscale : all;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = none ? 0.0f : rounded(v[i] * a);
    const int64_t e = n * D + c;
    if constexpr (OT == F32) {
      float* o = reinterpret_cast<float*>(out) + e;
      if (vec) *reinterpret_cast<float4*>(o) = float4{v[0], v[1], v[2], v[3]};
      else
        for (int i = 0; i < 4; ++i)
          if (c + i < D) o[i] = v[i];
    } else {
      uint16_t* o = reinterpret_cast<uint16_t*>(out) + e;
      const tg_u32x2 w = {tg_pack2<OT>(v[0], v[1]), tg_pack2<OT>(v[2], v[3])};
      if (vec) *reinterpret_cast<tg_u32x2*>(o) = w;
      else
        for (int i = 0; i < 4; ++i)
          if (c + i < D) o[i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
    }
  }
}

// --------------------------------------------------------------------------
// the plan of a call: what its shapes and types make of the workspace

struct LossPlan {
  int ct;            // the products' type
  int64_t dp;        // D in whole blocks of 64
  int64_t pitch;     // row pitch of the 16-bit copies
  bool copy_x, copy_w;
  int64_t piece;     // vocabulary rows a piece (a multiple of 256)
  int64_t vtiles;    // tiles of the vocabulary
  bool big_l, big_g;  // 256 x 256 tiles for the logits, the gradients
  int splits, wsplits;  // of grad_x's K, of grad_W's
  int lsplits;       // of the logits' K (1: their tiles are not stored)
  bool stream;       // forward: the table read as stored, for few tokens
  int64_t frag_bytes;
  size_t xc, wc, stats, tlogit, targets, each, scal, f, fx, fw, xs, P, sums, wsums, lsums, total;
};

// Time (us) of a round of tiles of 256 x 256 (a CU runs one workgroup of 8 waves) or
// of 128 x 128 (two of 4 waves) with K in blocks of 64.  Measured: the logits of 8192
// x 8192 at K 512 and 1024 take 85 and 131 us in 4 rounds of the first, 119 and 174
// in 8 of the second; those of 4096 x 16384 at K 4096 437 and 578, the gradients
// from them (512 blocks in 5 rounds, 1024 in 10) 916 and 1110.  A small tile that
// has its CU to itself takes 0.85 of the pair's time (2048 x 2048 and 2048 x 4096
// logits at K 1024: 20.6 and 24.3 us).
double round_us(bool big, double blocks, bool strided = false) {
  return big ? (strided ? 1.72 : 1.6) * blocks + 7.0 : 1.03 * blocks + 5.5;
}
constexpr double LONE = 0.85;

// Time of an M x N product of K.
double product_us(int64_t M, int64_t N, int64_t K, bool big) {
  const int64_t e = big ? 256 : 128, cus = device_cu_count();
  const int64_t tiles = ((M + e - 1) / e) * ((N + e - 1) / e);
  const double blocks = (double)((K + 63) / 64);
  const double round = round_us(big, blocks);
  if (big) return (double)((tiles + cus - 1) / cus) * round;
  const int64_t rest = tiles % (2 * cus);
  return (double)(tiles / (2 * cus)) * round +
         (rest == 0 ? 0.0 : rest <= cus ? LONE * round : round);
}
bool large_tiles(int64_t M, int64_t N, int64_t K) {
  return product_us(M, N, K, true) <= product_us(M, N, K, false);
}
double best_us(int64_t M, int64_t N, int64_t K) {
  return std::min(product_us(M, N, K, true), product_us(M, N, K, false));
}

// Both gradients' products in one launch: grad_x's tiles (K split) fill the
// workgroups' slots in rounds, grad_W's go where one is free first.
struct GradsPlan {
  double us;
  bool big;
  int splits, wsplits;
};
GradsPlan grads_plan(int64_t N, int64_t D, int64_t piece, int most = 64) {
  const int64_t cus = device_cu_count();
  GradsPlan best{0.0, false, 1, 1};
  const int64_t kx = (piece + 63) / 64, kw = (N + 63) / 64;
  for (int big = 0; big < 2; ++big) {
    const int64_t e = big ? 256 : 128, slots = big ? cus : 2 * cus, cols = (D + e - 1) / e;
    const int64_t nw = ((piece + e - 1) / e) * cols;
    // (grad_W's K, the tokens, is split where its tiles leave slots empty; each split's
    // sums cost a store, and a launch joins them.  The backward of 32768 x 512 x 256
    // classes: 120 us, unsplit 451; of 8192 x 1024 x 848, such as the last piece of
    // 50000 classes is: 103 and 159)
    for (int wsplits = 1; wsplits == 1 || (nw * wsplits <= 2 * slots && kw / wsplits >= 4);
         wsplits *= 2)
      for (int splits = 1; splits <= most && (splits == 1 || kx / splits >= 4); splits *= 2) {
        const int64_t nx = ((N + e - 1) / e) * cols * splits;
        const double tx = round_us(big != 0, (double)((kx + splits - 1) / splits), true);
        const double tw = round_us(big != 0, (double)((kw + wsplits - 1) / wsplits), true);
        // two groups of slots: those with one tile of grad_x more than the others
        int64_t count[2] = {nx % slots, slots - nx % slots}, left = nw * wsplits;
        double at[2] = {(double)(nx / slots + 1) * tx, (double)(nx / slots) * tx};
        double end = count[0] ? at[0] : at[1];
        while (left > 0) {
          const int g = count[0] == 0 || at[1] <= at[0] ? 1 : 0;
          at[g] += tw;
          end = std::max(end, at[g]);
          left -= count[g];
        }
        if (!big && nx + nw * wsplits <= cus) end *= LONE;
        // (the splits' sums: written and read once, a few at a time)
        double us = end + (double)splits * ((double)N * (double)D * 8.0 / 4e6 + 0.1);
        if (wsplits > 1) us += (double)wsplits * ((double)piece * (double)D * 8.0 / 4e6 + 0.1) + 5.0;
        if (best.us == 0.0 || us < best.us) best = GradsPlan{us, big != 0, splits, wsplits};
      }
  }
  return best;
}

// The splits of the logits' K where their tiles leave CUs idle, by the same model:
// each split's sums cost a store and a load, and a launch joins them (backward of
// 103 x 2560 x 1280 classes: 57 us, split 38; of 1 x 4096 x 1280: 67 and 33; forward
// of 300 x 4096 x 2000: 54 and 29).
int logit_splits(int64_t N, int64_t V, int64_t D, double* us) {
  const int64_t cus = device_cu_count(), blocks = (D + 63) / 64;
  const int64_t tiles = ((V + 127) / 128) * ((N + 127) / 128);
  *us = best_us(V, N, D);
  int best = 1;
  for (int s = 2; s <= 64 && blocks / s >= 2 && tiles * s <= 2 * cus; s *= 2) {
    const double round = round_us(false, (double)((blocks + s - 1) / s));
    const double t = (tiles * s <= cus ? LONE * round : round) + 5.0 +
                     s * ((double)N * (double)V * 8.0 / 4e6 + 0.3);
    if (t < *us) *us = t, best = s;
  }
  return best;
}

// The rows of a piece (a multiple of 256): at most 128 MiB of P (and of the
// table's 16-bit copy), so that what one product writes the next ones find in
// the 256 MB cache, but 1024 rows where the vocabulary has them (P of more than
// 65536 tokens is then larger: 2304 bytes a token); among the sizes that divide the vocabulary into about that
// many pieces, the one whose products take the least time by the model above.
int64_t loss_piece(int64_t N, int64_t D, int64_t dp, int64_t V, bool copy_w, bool backward) {
  const int64_t vr = (V + 255) / 256 * 256;
  int64_t most = vr;
  // (256 rows of P within 31 bits of bytes, whatever N)
  if (backward) most = std::min(most, ((int64_t)1 << 26) / std::max<int64_t>(N, 32));
  if (copy_w) most = std::min(most, ((int64_t)1 << 26) / dp);
  // (a launch's threads stay below 2^32: fewer than 2^24 tiles of 128 x 128, each 256)
  most = std::min(most, (((int64_t)1 << 24) - 1) / ((N + 127) / 128) * 128);
  most = std::max<int64_t>(most / 256 * 256, std::min<int64_t>(vr, 1024));
  if (most >= vr) return vr;
  auto cost = [&](int64_t rows) {
    if (rows == 0) return 0.0;
    double us = best_us(rows, N, D);
    if (!backward) return us + 5.0;
    logit_splits(N, rows, D, &us);
    return us + grads_plan(N, D, rows).us + 10.0;
  };
  int64_t best = most;
  double least = 0.0;
  const int64_t few = (vr + most - 1) / most;
  for (int64_t k = few; k < few + 6; ++k) {
    // k equal pieces, or whole ones of `most` first (k == few)
    for (int whole = 0; whole < 2; ++whole) {
      const int64_t rows = whole ? most : ((V + k - 1) / k + 255) / 256 * 256;
      if (rows > most) continue;
      const double us = (double)(V / rows) * cost(rows) + cost(V % rows);
      if (least == 0.0 || us < least) least = us, best = rows;
    }
  }
  return best;
}

int stream_tiles(int64_t N) { return N <= 32 ? 1 : N <= 64 ? 2 : 4; }

LossPlan loss_plan(int64_t N, int64_t D, int64_t V, int x_dtype, int w_dtype, bool backward) {
  LossPlan p{};
  p.ct = x_dtype == F16 ? F16 : BF16;
  p.dp = (D + 63) / 64 * 64;
  p.pitch = row_pitch(p.dp);
  // x is copied in the backward (ignored rows become zeros, which its product
  // over the rows needs) and where it is not in the products' type and whole
  // blocks of 64
  p.copy_x = backward || x_dtype != p.ct || D % 64 != 0;
  p.copy_w = w_dtype != p.ct || D % 64 != 0;
  p.piece = loss_piece(N, D, p.dp, V, p.copy_w, backward);
  p.big_l = large_tiles(p.piece, N, D);
  p.vtiles = (V + (p.big_l ? 255 : 127)) / (p.big_l ? 256 : 128);
  double logits_us = 0.0;
  // (the forward's rows are joined from one piece)
  p.lsplits = 1;
  if (backward || p.piece >= V) p.lsplits = logit_splits(N, std::min(p.piece, V), D, &logits_us);
  // up to 128 rows of x, codes whose rows are whole 16-byte chunks, in a type that
  // the kernel decodes (16-bit ones as they are)
  p.stream = !backward && N <= 128 && row_bytes(w_dtype, D) % 16 == 0 &&
             (is_quant(w_dtype) || w_dtype == p.ct);
  if (p.stream) {
    const int E = 128 / dtype_bits(w_dtype), nt = stream_tiles(N);
    // a small table's few workgroups take their stages one after another, each the
    // longer the more fragments it copies: 0.54 us for one tile of tokens with E4M3
    // codes, 1.6 for four, 2.9 with E2M1 ones; the split logits have a copy of the
    // table in place of a join, taken as 2 us less than the model's.  GPU time of a
    // call so and split: 103 tokens of 2560, 1280 classes E4M3 43.9 and 19.9 us; 37 of
    // 4096, 5000 E2M1 39.4 and 34.1; 1 of 4096, 5000 E4M3 23.8 and 33.6; 16 of 4096,
    // 2000 E2M1 22.0 and 23.0.  Of 108 shapes (1 to 128 tokens of 1024 to 8192, 512 to
    // 5000 classes, E4M3, E2M1, bf16) the rule takes the faster side for 83 and loses
    // at most 11 us on the others (64 of 2560, 1280 classes E2M1: 28.9 us, split 18.4;
    // 128 of 1024, 1000 classes E4M3: 23.8 and 16.3).
    const int64_t stages = (D + 8 * E - 1) / (8 * E);
    if (p.lsplits > 1 && (double)stages * (0.2 + 0.17 * (E / 8) * nt) > logits_us - 2.0)
      p.stream = false;
    else p.lsplits = 1;
  }
  if (p.stream) {
    const int E = 128 / dtype_bits(w_dtype), nt = stream_tiles(N);
    p.frag_bytes = ((D + 8 * E - 1) / (8 * E)) * 4 * (E / 8) * nt * 1024;
    p.big_l = p.copy_x = p.copy_w = false;
    p.vtiles = (V + stream_rows(E, nt) - 1) / stream_rows(E, nt);
  }
  if (backward) {
    const GradsPlan g = grads_plan(N, D, p.piece);
    p.big_g = g.big;
    p.splits = g.splits;
    p.wsplits = g.wsplits;
  }
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t b = at;
    at += align256(bytes);
    return b;
  };
  p.targets = take((size_t)N * 4);
  p.scal = take(16);
  p.xc = take(p.stream ? (size_t)p.frag_bytes : p.copy_x ? (size_t)N * p.pitch * 2 : 0);
  p.wc = take(p.copy_w ? (size_t)p.piece * p.pitch * 2 : 0);
  auto logit_parts = [&](int splits, int64_t rows) {
    return splits > 1 ? (size_t)splits * N * ((rows + 255) / 256 * 256) * 4 : 0;
  };
  size_t lparts = logit_parts(p.lsplits, std::min(p.piece, V));
  if (backward && V > p.piece && V % p.piece)
    lparts = std::max(lparts, logit_parts(logit_splits(N, V % p.piece, D, &logits_us), V % p.piece));
  p.lsums = take(lparts);
  if (backward) {
    p.f = take((size_t)N * 4);
    p.fx = take((size_t)N * 4);  // (these three where each row has a gradient of its own)
    p.fw = take((size_t)N * 4);
    p.xs = take((size_t)N * p.pitch * 2);
    p.P = take((size_t)N * row_pitch(p.piece) * 2);
    p.sums = take((size_t)p.splits * N * p.dp * 4);
    auto parts = [&](int splits, int64_t rows) {
      return splits > 1 ? (size_t)splits * rows * p.dp * 4 : 0;
    };
    const int64_t rest = V % p.piece;
    const size_t last =
        V > p.piece && rest ? parts(grads_plan(N, D, rest, p.splits).wsplits, rest) : 0;
    p.wsums = take(std::max(parts(p.wsplits, std::min(p.piece, V)), last));
  } else {
    p.stats = take((size_t)N * p.vtiles * 8);
    p.tlogit = take((size_t)N * 4);
    p.each = take((size_t)N * 4);
  }
  p.total = at;
  return p;
}

template <class G>
int raise_lds(const void* kern, DeviceFlags& raised) {
  return allow_lds(raised, kern, G::lds_bytes, G::lds_bytes);
}

#define NOVAQ_LAUNCH(KERN, GRID, G, STREAM, ...)                                          \
  do {                                                                                    \
    static DeviceFlags raised;                                                            \
    const int rc_ = raise_lds<G>(reinterpret_cast<const void*>(&KERN), raised);           \
    if (rc_ != NOVAQ_OK) return rc_;                                                      \
    hipLaunchKernelGGL(KERN, dim3((unsigned)(GRID)), dim3(G::NTH), G::lds_bytes, STREAM,  \
                       __VA_ARGS__);                                                      \
    const int rl_ = check_launch();                                                       \
    if (rl_ != NOVAQ_OK) return rl_;                                                      \
  } while (0)

template <int CT>
int stream(const LossPlan& p, int64_t N, int64_t D, const void* w, int w_dtype,
           const float* w_scale, int64_t V, const int* targets, float2* stats, float* tl,
           const uint16_t* frags, hipStream_t st) {
  const int nt = stream_tiles(N);
  auto go = [&](auto wt, auto tiles) -> int {
    constexpr int WT = decltype(wt)::value;
    using S = TokenStream<CT, WT, decltype(tiles)::value>;
    NOVAQ_LAUNCH((loss_stream_kernel<CT, WT, S>), p.vtiles, S, st, static_cast<const uint8_t*>(w),
                 V, row_bytes(w_dtype, D), reinterpret_cast<const uint8_t*>(frags),
                 S::kstages(D), w_scale, N, targets, stats, p.vtiles, tl);
    return NOVAQ_OK;
  };
  auto to = [&](auto wt) -> int {
    return nt == 1   ? go(wt, std::integral_constant<int, 1>{})
           : nt == 2 ? go(wt, std::integral_constant<int, 2>{})
                     : go(wt, std::integral_constant<int, 4>{});
  };
  switch (w_dtype) {
    case E4M3: return to(std::integral_constant<int, E4M3>{});
    case E5M2: return to(std::integral_constant<int, E5M2>{});
    case E2M1: return to(std::integral_constant<int, E2M1>{});
    default: return to(std::integral_constant<int, CT>{});
  }
}

template <int CT>
int logits(const LossPlan& p, int splits, const TokenOp& ow, const TokenOp& ox, int64_t N,
           uint8_t* ws, hipStream_t st) {
  using G = TokenGemm<CT, false, false, 64, 64, 2>;
  const int tm = (int)((ow.rows + G::BM - 1) / G::BM), tn = (int)((N + G::BN - 1) / G::BN);
  NOVAQ_LAUNCH((loss_logits_kernel<CT, G>), (int64_t)tm * tn * splits, G, st, ow, ox, p.dp, N,
               splits, reinterpret_cast<float*>(ws + p.lsums), (ow.rows + 255) / 256 * 256, tm,
               tn);
  return NOVAQ_OK;
}

template <int CT>
int forward(const LossPlan& p, const void* x, int x_dtype, int64_t N, int64_t D, const void* w,
            int w_dtype, const float* w_scale, int64_t V, const void* ids, int bits,
            int64_t ignore, int reduction, float* loss, float* lse, uint8_t* ws, hipStream_t st) {
  int* targets = reinterpret_cast<int*>(ws + p.targets);
  float* scal = reinterpret_cast<float*>(ws + p.scal);
  float2* stats = reinterpret_cast<float2*>(ws + p.stats);
  float* tl = reinterpret_cast<float*>(ws + p.tlogit);
  float* each = reduction == NOVAQ_REDUCE_NONE ? loss : reinterpret_cast<float*>(ws + p.each);
  uint16_t* xw = reinterpret_cast<uint16_t*>(ws + p.xc);
  uint16_t* ww = reinterpret_cast<uint16_t*>(ws + p.wc);
  RowsJob rows{ids, bits, ignore, N, V, nullptr, 0, 0, targets, nullptr, scal, nullptr, nullptr};
  CopyJob cx{};
  FragmentJob fx{};
  if (p.stream)
    fx = FragmentJob{static_cast<const uint8_t*>(x), xw, N, D, p.frag_bytes / 16, x_dtype,
                     128 / dtype_bits(w_dtype), stream_tiles(N)};
  else if (p.copy_x)
    cx = CopyJob{static_cast<const uint8_t*>(x), xw, N, D, p.dp, p.pitch, x_dtype, nullptr, 0, 0, {}};
  int rc = NOVAQ_OK;
  if (p.stream) {
    rc = prep_launch<CT>(rows, cx, fx, CopyJob{}, st);
    if (rc == NOVAQ_OK) rc = stream<CT>(p, N, D, w, w_dtype, w_scale, V, targets, stats, tl, xw, st);
    if (rc != NOVAQ_OK) return rc;
  }
  const TokenOp ox{p.copy_x ? xw : static_cast<const uint16_t*>(x), N, p.copy_x ? p.pitch : D};
  for (int64_t v0 = 0; v0 < V && !p.stream; v0 += p.piece) {
    const int64_t vc = std::min(p.piece, V - v0);
    const uint8_t* from = static_cast<const uint8_t*>(w) + v0 * row_bytes(w_dtype, D);
    CopyJob cw{};
    if (p.copy_w) cw = CopyJob{from, ww, vc, D, p.dp, p.pitch, w_dtype, nullptr, 0, 0, {}};
    rc = prep_launch<CT>(rows, cx, fx, cw, st);
    if (rc != NOVAQ_OK) return rc;
    rows.N = cx.rows = 0;  // (done with the first piece)
    const TokenOp ow{p.copy_w ? ww : reinterpret_cast<const uint16_t*>(from), vc,
                     p.copy_w ? p.pitch : D};
    if (p.lsplits > 1) {
      rc = logits<CT>(p, p.lsplits, ow, ox, N, ws, st);
      if (rc != NOVAQ_OK) return rc;
      hipLaunchKernelGGL(loss_rows_kernel, dim3((unsigned)N), dim3(256), 0, st,
                         reinterpret_cast<const float*>(ws + p.lsums), p.lsplits, N, V,
                         (V + 255) / 256 * 256, w_scale, targets, lse, each);
      rc = check_launch();
      if (rc != NOVAQ_OK) return rc;
      break;
    }
    auto stats_of = [&](auto g) -> int {
      using G = decltype(g);
      const int tm = (int)((vc + G::BM - 1) / G::BM), tn = (int)((N + G::BN - 1) / G::BN);
      NOVAQ_LAUNCH((loss_stats_kernel<CT, G>), (int64_t)tm * tn, G, st, ow, ox, p.dp, w_scale,
                   v0, N, targets, stats, p.vtiles, tl, tm, tn);
      return NOVAQ_OK;
    };
    rc = p.big_l ? stats_of(TokenGemm<CT, false, false, 128, 64, 4>{})
                 : stats_of(TokenGemm<CT, false, false, 64, 64, 2>{});
    if (rc != NOVAQ_OK) return rc;
  }
  float* out = reduction == NOVAQ_REDUCE_NONE ? nullptr : loss;
  bool alone = false;
  if (p.lsplits == 1) {
    // (one workgroup, that sums the losses too, for up to 16 rows; the 37 of 1024 x
    // 50000 take 23.5 us a call so, with a workgroup for 16 rows each 20.0)
    alone = N <= 16;
    hipLaunchKernelGGL(loss_join_kernel,
                       dim3(alone ? 1u : (unsigned)std::min<int64_t>((N + 15) / 16, 1 << 18)),
                       dim3(1024), 0, st, stats, p.vtiles, N, targets, tl, lse, each,
                       reduction == NOVAQ_REDUCE_MEAN, scal, out);
    rc = check_launch();
  }
  if (rc != NOVAQ_OK || alone || !out) return rc;
  hipLaunchKernelGGL(loss_sum_kernel, dim3(1), dim3(1024), 0, st, each, N,
                     reduction == NOVAQ_REDUCE_MEAN, scal, out);
  return check_launch();
}

template <int OT>
int store_sums(const float* sums, int splits, int64_t rows, int64_t dp, int64_t D,
               const float* scal, const float* w_scale, float inv, const int* targets,
               const float* fx, void* out, hipStream_t st) {
  auto go = [&](auto share) {
    constexpr bool SHARE = decltype(share)::value;
    const int64_t units = SHARE ? 64 : 256;
    const dim3 grid((unsigned)std::min<int64_t>((rows * (dp / 4) + units - 1) / units, 8192));
    hipLaunchKernelGGL((loss_sums_store_kernel<OT, SHARE>), grid, dim3(256), 0, st, sums, splits,
                       rows, dp, D, scal, w_scale, inv, targets, fx, out);
  };
  if (splits >= 8) go(std::true_type{});
  else go(std::false_type{});
  return check_launch();
}

template <int CT>
int backward(const LossPlan& p, const void* x, int x_dtype, int64_t N, int64_t D, const void* w,
             int w_dtype, const float* w_scale, int64_t V, const void* ids, int bits,
             int64_t ignore, int reduction, const float* grad, const float* lse, void* gx,
             void* gw, int gw_dtype, uint8_t* ws, hipStream_t st) {
  int* targets = reinterpret_cast<int*>(ws + p.targets);
  float* scal = reinterpret_cast<float*>(ws + p.scal);
  float* f = reinterpret_cast<float*>(ws + p.f);
  uint16_t* P = reinterpret_cast<uint16_t*>(ws + p.P);
  float* sums = reinterpret_cast<float*>(ws + p.sums);
  uint16_t* xw = reinterpret_cast<uint16_t*>(ws + p.xc);
  uint16_t* ww = reinterpret_cast<uint16_t*>(ws + p.wc);
  const float pscale = CT == F16 ? 0x1p14f : 1.0f, inv = 1.0f / pscale;
  const bool per_row = reduction == NOVAQ_REDUCE_NONE && grad;
  float* fx = reinterpret_cast<float*>(ws + p.fx);
  float* fw = reinterpret_cast<float*>(ws + p.fw);
  uint16_t* xs = reinterpret_cast<uint16_t*>(ws + p.xs);
  RowsJob rows{ids, bits, ignore, N, V, grad, per_row ? 1 : 0, reduction == NOVAQ_REDUCE_MEAN,
               targets, f, scal, fx, fw};
  CopyJob cx{static_cast<const uint8_t*>(x), xw, N, D, p.dp, p.pitch, x_dtype, ids, bits, ignore, {}};
  int rc = NOVAQ_OK;
  const TokenOp ox{xw, N, p.pitch}, oxs{per_row && gw ? xs : xw, N, p.pitch};
  for (int64_t v0 = 0; v0 < V; v0 += p.piece) {
    const int64_t vc = std::min(p.piece, V - v0), vp = (vc + 255) / 256 * 256;
    const uint8_t* from = static_cast<const uint8_t*>(w) + v0 * row_bytes(w_dtype, D);
    CopyJob cw{};
    if (p.copy_w) cw = CopyJob{from, ww, vc, D, p.dp, p.pitch, w_dtype, nullptr, 0, 0, {}};
    rc = prep_launch<CT>(rows, cx, FragmentJob{}, cw, st);
    if (rc != NOVAQ_OK) return rc;
    rows.N = cx.rows = 0;  // (done with the first piece)
    if (per_row && gw && v0 == 0) {
      const dim3 grid((unsigned)std::min<int64_t>((N * (p.dp / 8) + 255) / 256, 8192));
      hipLaunchKernelGGL(loss_scaled_x_kernel<CT>, grid, dim3(256), 0, st, xw, fw, N, p.dp, p.pitch,
                         xs);
      rc = check_launch();
      if (rc != NOVAQ_OK) return rc;
    }
    const int64_t pp = row_pitch(vp);
    const TokenOp ow{p.copy_w ? ww : reinterpret_cast<const uint16_t*>(from), vc,
                     p.copy_w ? p.pitch : D};
    // a last, smaller piece may do better on other tiles (the first has set all the
    // splits' sums)
    const bool rest = v0 > 0 && vc < p.piece;
    const bool big_l = rest ? large_tiles(vc, N, D) : p.big_l;
    const GradsPlan gp = rest ? grads_plan(N, D, vc, p.splits)
                              : GradsPlan{0.0, p.big_g, p.splits, p.wsplits};
    auto prob = [&](auto g) -> int {
      using G = decltype(g);
      const int tm = (int)(vp / G::BM), tn = (int)((N + G::BN - 1) / G::BN);
      NOVAQ_LAUNCH((loss_prob_kernel<CT, G>), (int64_t)tm * tn, G, st, ow, ox, p.dp, w_scale, v0,
                   N, targets, f, lse, pscale, P, pp, tm, tn);
      return NOVAQ_OK;
    };
    double us;
    const int lsplits = rest ? logit_splits(N, vc, D, &us) : p.lsplits;
    if (lsplits > 1) {
      rc = logits<CT>(p, lsplits, ow, ox, N, ws, st);
      if (rc != NOVAQ_OK) return rc;
      hipLaunchKernelGGL(loss_prob_rows_kernel<CT>, dim3((unsigned)((vp + 2047) / 2048), (unsigned)N),
                         dim3(256), 0, st, reinterpret_cast<const float*>(ws + p.lsums), lsplits, N,
                         vc, vp, v0, w_scale, targets, f, lse, pscale, P, pp);
      rc = check_launch();
    } else {
      rc = big_l ? prob(TokenGemm<CT, false, false, 128, 64, 4>{})
                 : prob(TokenGemm<CT, false, false, 64, 64, 2>{});
    }
    if (rc != NOVAQ_OK) return rc;
    auto grads = [&](auto ot, auto gx_, auto gw_) -> int {
      using GX = decltype(gx_);
      using GW = decltype(gw_);
      constexpr int OT = decltype(ot)::value;
      GradsJob j{TokenOp{P, N, pp}, TokenOp{P, vp, pp}, ow, oxs, N, D, vc, (int)(vp / 64),
                 (int)((N + 63) / 64), gp.splits, v0 == 0 ? 1 : 0, sums, p.dp, scal, inv,
                 static_cast<uint8_t*>(gw) + v0 * D * (OT == F32 ? 4 : 2),
                 reinterpret_cast<float*>(ws + p.wsums), gp.wsplits, 0, 0, 0, 0};
      if (gx) {
        j.xtm = (int)((N + GX::BM - 1) / GX::BM);
        j.xtn = (int)((D + GX::BN - 1) / GX::BN);
      } else {
        j.xtm = j.xtn = 0;
      }
      if (gw) {
        j.wtm = (int)((vc + GW::BM - 1) / GW::BM);
        j.wtn = (int)((D + GW::BN - 1) / GW::BN);
      }
      const int64_t tiles = (int64_t)j.xtm * j.xtn * j.splits + (int64_t)j.wtm * j.wtn * j.wsplits;
      if (!gw || gp.wsplits == 1) {
        NOVAQ_LAUNCH((loss_grads_kernel<CT, OT, GX, GW>), tiles, GX, st, j);
        return NOVAQ_OK;
      }
      NOVAQ_LAUNCH((loss_grads_kernel<CT, SUMS, GX, GW>), tiles, GX, st, j);
      return store_sums<OT>(j.wsums, gp.wsplits, vc, p.dp, D, scal, nullptr, inv, nullptr, nullptr, j.gw,
                            st);
    };
    auto grads_to = [&](auto ot) -> int {
      return gp.big ? grads(ot, TokenGemm<CT, false, true, 128, 64, 4>{},
                             TokenGemm<CT, true, true, 128, 64, 4>{})
                     : grads(ot, TokenGemm<CT, false, true, 64, 64, 2>{},
                             TokenGemm<CT, true, true, 64, 64, 2>{});
    };
    rc = gw_dtype == F32   ? grads_to(std::integral_constant<int, F32>{})
         : gw_dtype == F16 ? grads_to(std::integral_constant<int, F16>{})
                           : grads_to(std::integral_constant<int, BF16>{});
    if (rc != NOVAQ_OK) return rc;
  }
  if (!gx) return rc;
  auto store = [&](auto ot) {
    return store_sums<decltype(ot)::value>(sums, p.splits, N, p.dp, D, scal, w_scale, inv, targets,
                                           per_row ? fx : nullptr, gx, st);
  };
  return x_dtype == F32   ? store(std::integral_constant<int, F32>{})
         : x_dtype == F16 ? store(std::integral_constant<int, F16>{})
                          : store(std::integral_constant<int, BF16>{});
}

#undef NOVAQ_LAUNCH

}  // namespace

size_t vocab_loss_workspace(int64_t N, int64_t D, int64_t V, int x_dtype, int w_dtype,
                            bool backward) {
  return loss_plan(N, D, V, x_dtype, w_dtype, backward).total;
}

int vocab_loss_launch(const void* x, int x_dtype, int64_t N, int64_t D, const void* w, int w_dtype,
                      const float* w_scale, int64_t V, const void* ids, int bits, int64_t ignore,
                      int reduction, float* loss, float* lse, void* ws, hipStream_t stream) {
  const LossPlan p = loss_plan(N, D, V, x_dtype, w_dtype, false);
  uint8_t* b = static_cast<uint8_t*>(ws);
  return p.ct == F16 ? forward<F16>(p, x, x_dtype, N, D, w, w_dtype, w_scale, V, ids, bits, ignore,
                                    reduction, loss, lse, b, stream)
                     : forward<BF16>(p, x, x_dtype, N, D, w, w_dtype, w_scale, V, ids, bits,
                                     ignore, reduction, loss, lse, b, stream);
}

int vocab_loss_backward_launch(const void* x, int x_dtype, int64_t N, int64_t D, const void* w,
                               int w_dtype, const float* w_scale, int64_t V, const void* ids,
                               int bits, int64_t ignore, int reduction, const float* grad,
                               const float* lse, void* gx, void* gw, int gw_dtype, void* ws,
                               hipStream_t stream) {
  const LossPlan p = loss_plan(N, D, V, x_dtype, w_dtype, true);
  uint8_t* b = static_cast<uint8_t*>(ws);
  return p.ct == F16
             ? backward<F16>(p, x, x_dtype, N, D, w, w_dtype, w_scale, V, ids, bits, ignore,
                             reduction, grad, lse, gx, gw, gw_dtype, b, stream)
             : backward<BF16>(p, x, x_dtype, N, D, w, w_dtype, w_scale, V, ids, bits, ignore,
                              reduction, grad, lse, gx, gw, gw_dtype, b, stream);
}

}  // namespace novaq
