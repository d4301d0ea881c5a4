// Embedding lookup in a table of any stored type, and its gradient by sorted
// tokens.
//
//   out[i]     = dec(W[t[i]]) * (s * factor)
//   grad_W[v] (+)= factor * sum over i with t[i] = v of grad[i]
//
// The lookup moves one row a token and is bound by memory; 8 elements a lane.
//
// The gradient sorts the tokens (stable, radix digits of 9 bits), so that a
// row's positions lie together in rising order, and sums runs of 16 sorted
// entries a wave.  A token with many positions spans several of these chunks:
// each then leaves its part in the workspace and a last kernel adds a run's
// parts in order.  No atomics touch floating-point values: the sums' order
// depends on the tokens alone, and the result is the same bit for bit in every
// call.  Sums are fp32; the factor is applied once to the whole sum.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "novaq_internal.h"
#include "token_io.h"

namespace novaq {
namespace {

// A row per token, 8 elements a thread; a token outside the table gives a row
// of NaN.
template <int ST, int OT, bool VEC>
__global__ __launch_bounds__(256) void embedding_kernel(const void* __restrict__ ids, int bits,
                                                        int64_t N,
                                                        const uint8_t* __restrict__ table,
                                                        const float* __restrict__ scale,
                                                        int64_t V, int64_t D, float factor,
                                                        void* __restrict__ out) {
  const int64_t per = (D + 7) / 8, rb = row_bytes(ST, D);
  const float a = (scale ? *scale : 1.0f) * factor;
  for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < N * per;
       q += (int64_t)gridDim.x * 256) {
    const int64_t i = q / per, c = (q - i * per) * 8;
    const int64_t t = token_at(ids, bits, i);
    float v[8];
    if (t >= 0 && t < V) {
      load8<ST, VEC>(table + t * rb, c, D, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= a;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = u2f(0x7FC00000u);
    }
    store8<OT, VEC>(out, i * D + c, D - c, v);
  }
}

template <int ST, int OT>
int lookup(const void* ids, int bits, int64_t N, const void* table, const float* scale, int64_t V,
           int64_t D, float factor, void* out, hipStream_t st) {
  const int64_t units = N * ((D + 7) / 8);
  const dim3 grid((unsigned)std::min<int64_t>((units + 255) / 256, 1 << 20));
  const uint8_t* t = static_cast<const uint8_t*>(table);
  if (D % 8 == 0)
    hipLaunchKernelGGL((embedding_kernel<ST, OT, true>), grid, dim3(256), 0, st, ids, bits, N, t,
                       scale, V, D, factor, out);
  else
    hipLaunchKernelGGL((embedding_kernel<ST, OT, false>), grid, dim3(256), 0, st, ids, bits, N, t,
                       scale, V, D, factor, out);
  return check_launch();
}

template <int ST>
int lookup_to(int ot, const void* ids, int bits, int64_t N, const void* table, const float* scale,
              int64_t V, int64_t D, float factor, void* out, hipStream_t st) {
  switch (ot) {
    case F32: return lookup<ST, F32>(ids, bits, N, table, scale, V, D, factor, out, st);
    case F16: return lookup<ST, F16>(ids, bits, N, table, scale, V, D, factor, out, st);
    case BF16: return lookup<ST, BF16>(ids, bits, N, table, scale, V, D, factor, out, st);
    default: return NOVAQ_EDTYPE;
  }
}

// --------------------------------------------------------------------------
// the sort

constexpr int DIGIT = 9, BINS = 1 << DIGIT;
constexpr int BLOCKS = 128;     // at most, of a pass
constexpr int CHUNK = 16;       // sorted entries a wave sums

// The sort's key of position i: the token, or V where it is none of the
// table's (those sort last and are left out).
__device__ __forceinline__ uint32_t token_key(const void* ids, int bits, int64_t i, int64_t V) {
  const int64_t t = token_at(ids, bits, i);
  return t >= 0 && t < V ? (uint32_t)t : (uint32_t)V;
}

// Digit counts of each block's `per` entries: hist[block][digit].
__global__ __launch_bounds__(256) void sort_hist_kernel(const uint32_t* __restrict__ keys,
                                                        const void* __restrict__ ids, int bits,
                                                        int64_t V, int N, int per, int shift,
                                                        uint32_t* __restrict__ hist) {
  __shared__ uint32_t cnt[BINS];
  for (int d = threadIdx.x; d < BINS; d += 256) cnt[d] = 0;
  __syncthreads();
  const int from = blockIdx.x * per, to = min(N, from + per);
  for (int i = from + threadIdx.x; i < to; i += 256) {
    const uint32_t k = ids ? token_key(ids, bits, i, V) : keys[i];
    atomicAdd(&cnt[(k >> shift) & (BINS - 1)], 1u);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < BINS; d += 256) hist[blockIdx.x * BINS + d] = cnt[d];
}

// One stable pass: entry i of digit d goes behind all entries of smaller
// digits, those of d in earlier blocks, and those of d before it in its block.
// Each wave takes a contiguous quarter of the block, 64 entries a step; equal
// digits within a step are ranked by ballots.
__global__ __launch_bounds__(256) void sort_scatter_kernel(
    const uint32_t* __restrict__ keys, const uint32_t* __restrict__ pos,
    const void* __restrict__ ids, int bits, int64_t V, int N, int per, int shift,
    const uint32_t* __restrict__ hist, uint32_t* __restrict__ keys_out,
    uint32_t* __restrict__ pos_out) {
  __shared__ uint32_t base[BINS], cnt[4][BINS], sums[256];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int nb = gridDim.x, b = blockIdx.x;
  // digits 2 tid and 2 tid + 1: entries of earlier blocks, and of all
  uint32_t before[2] = {0, 0}, all[2] = {0, 0};
#pragma unroll 8
  for (int i = 0; i < nb; ++i) {
    const uint2 h = reinterpret_cast<const uint2*>(hist + i * BINS)[tid];
    all[0] += h.x, all[1] += h.y;
    if (i < b) before[0] += h.x, before[1] += h.y;
  }
  sums[tid] = all[0] + all[1];
  for (int w = 0; w < 4; ++w) cnt[w][2 * tid] = 0, cnt[w][2 * tid + 1] = 0;
  __syncthreads();
  for (int d = 1; d < 256; d <<= 1) {
    const uint32_t o = tid >= d ? sums[tid - d] : 0;
    __syncthreads();
    sums[tid] += o;
    __syncthreads();
  }
  const uint32_t first = sums[tid] - all[0] - all[1];
  base[2 * tid] = first + before[0];
  base[2 * tid + 1] = first + all[0] + before[1];
  // the waves' own counts
  const int quarter = per / 4, from = b * per + wave * quarter,
            to = min(N, from + quarter);
  for (int i = from + lane; i < to; i += 64) {
    const uint32_t k = ids ? token_key(ids, bits, i, V) : keys[i];
    atomicAdd(&cnt[wave][(k >> shift) & (BINS - 1)], 1u);
  }
  __syncthreads();
  for (int d = tid; d < BINS; d += 256) {
    uint32_t at = base[d];
    for (int w = 0; w < 4; ++w) {
      const uint32_t c = cnt[w][d];
      cnt[w][d] = at;
      at += c;
    }
  }
  __syncthreads();
  for (int i0 = from; i0 < to; i0 += 64) {
    const int i = i0 + lane;
    const bool in = i < to;
    uint32_t k = 0, p = 0;
    if (in) {
      k = ids ? token_key(ids, bits, i, V) : keys[i];
      p = ids ? (uint32_t)i : pos[i];
    }
    const uint32_t d = (k >> shift) & (BINS - 1);
    uint64_t same = __ballot(in);
#pragma unroll
    for (int bit = 0; bit < DIGIT; ++bit) {
      const uint64_t m = __ballot((d >> bit) & 1);
      same &= (d >> bit) & 1 ? m : ~m;
    }
    const uint32_t rank = __popcll(same & ((1ull << lane) - 1));
    uint32_t at = 0;
    if (in) at = cnt[wave][d] + rank;
    // (the reads above come before the first lane's write, the next step's after)
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (in && rank == 0) cnt[wave][d] += (uint32_t)__popcll(same);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (in) {
      keys_out[at] = k;
      pos_out[at] = p;
    }
  }
}

// --------------------------------------------------------------------------
// the sums

// VEC elements from p as fp32 (VEC 8: 16-byte loads; 4: one load).
template <int GT, int VEC>
__device__ __forceinline__ void loadv(const uint8_t* p, float (&v)[VEC]) {
  if constexpr (VEC == 8) {
    load8<GT, true>(p, 0, 8, v);
  } else if constexpr (VEC == 4) {
    if constexpr (GT == F32) {
      const ti_u32x4 a = *reinterpret_cast<const ti_u32x4*>(p);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = u2f(a[i]);
    } else {
      const ti_u32x2 a = *reinterpret_cast<const ti_u32x2*>(p);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t w = a[i];
        v[2 * i] = u2f(decode<GT>(w & 0xFFFFu));
        v[2 * i + 1] = u2f(decode<GT>(w >> 16));
      }
    }
  } else {
    if constexpr (GT == F32) v[0] = *reinterpret_cast<const float*>(p);
    else v[0] = u2f(decode<GT>(*reinterpret_cast<const uint16_t*>(p)));
  }
}

template <int OT, int VEC>
__device__ __forceinline__ void storev(uint8_t* p, const float (&v)[VEC]) {
  if constexpr (VEC == 8) {
    store8<OT, true>(p, 0, 8, v);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      if constexpr (OT == F32) reinterpret_cast<float*>(p)[i] = v[i];
      else reinterpret_cast<uint16_t*>(p)[i] = (uint16_t)encode<OT>(f2u(v[i]));
    }
  }
}

template <int OT, int VEC>
__device__ __forceinline__ void put_row(uint8_t* out, const float (&sum)[VEC], float factor,
                                        int accumulate) {
  float y[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) y[i] = sum[i] * factor;
  if (accumulate) {
    float old[VEC];
    loadv<OT, VEC>(out, old);
#pragma unroll
    for (int i = 0; i < VEC; ++i) y[i] += old[i];
  }
  storev<OT, VEC>(out, y);
}

// One wave: a chunk of sorted entries x 64 VEC columns.  All rows are loaded
// before the first sum; a run that ends inside the chunk is stored, one that
// began in an earlier chunk leaves its sum at head[chunk], one that goes on
// past the chunk at tail[chunk].
template <int GT, int OT, int VEC>
__global__ __launch_bounds__(256) void embedding_sum_kernel(
    const uint8_t* __restrict__ grad, const uint32_t* __restrict__ keys,
    const uint32_t* __restrict__ pos, int N, int64_t V, int64_t D, float factor, int accumulate,
    float* __restrict__ head, float* __restrict__ tail, uint8_t* __restrict__ out) {
  constexpr int GB = GT == F32 ? 4 : 2, OB = OT == F32 ? 4 : 2;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int chunk = blockIdx.x * 4 + wave, lane = threadIdx.x & 63;
  const int e0 = chunk * CHUNK, n = min(CHUNK, N - e0);
  if (n <= 0) return;
  const int64_t c = (int64_t)blockIdx.y * 64 * VEC + lane * VEC;
  if (c >= D) return;
  float v[CHUNK][VEC];
  uint32_t k[CHUNK];
#pragma unroll
  for (int i = 0; i < CHUNK; ++i) {
    const int e = e0 + min(i, n - 1);
    k[i] = keys[e];
    loadv<GT, VEC>(grad + ((int64_t)pos[e] * D + c) * GB, v[i]);
  }
  const bool from_before = chunk > 0 && keys[e0 - 1] == k[0];
  const bool goes_on = e0 + n < N && keys[e0 + n] == k[n - 1];
  float sum[VEC];
#pragma unroll
  for (int x = 0; x < VEC; ++x) sum[x] = 0.0f;
  bool at_start = true;
#pragma unroll
  for (int i = 0; i < CHUNK; ++i) {
    if (i < n) {
#pragma unroll
      for (int x = 0; x < VEC; ++x) sum[x] += v[i][x];
      const bool last = i == n - 1;
      if (last || k[i < CHUNK - 1 ? i + 1 : i] != k[i]) {
        if ((int64_t)k[i] < V) {
          if (at_start && from_before)
            storev<F32, VEC>(reinterpret_cast<uint8_t*>(head + (int64_t)chunk * D + c), sum);
          else if (last && goes_on)
            storev<F32, VEC>(reinterpret_cast<uint8_t*>(tail + (int64_t)chunk * D + c), sum);
          else
            put_row<OT, VEC>(out + ((int64_t)k[i] * D + c) * OB, sum, factor, accumulate);
        }
        at_start = false;
#pragma unroll
        for (int x = 0; x < VEC; ++x) sum[x] = 0.0f;
      }
    }
  }
}

// The runs that span chunks: the chunk where one begins adds its tail and the
// heads of the chunks after it.  Eight waves take every eighth head each; their
// sums are added in the waves' order.
template <int OT, int VEC>
__global__ __launch_bounds__(512) void embedding_join_kernel(
    const uint32_t* __restrict__ keys, int N, int64_t V, int64_t D, float factor, int accumulate,
    const float* __restrict__ head, const float* __restrict__ tail, uint8_t* __restrict__ out) {
  constexpr int OB = OT == F32 ? 4 : 2;
  __shared__ float part[8][64 * VEC];
  const int chunk = blockIdx.x, lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int e0 = chunk * CHUNK, e1 = e0 + CHUNK;
  if (e1 >= N) return;
  const uint32_t k = keys[e1 - 1];
  if (keys[e1] != k || (int64_t)k >= V) return;
  if (e0 > 0 && keys[e0] == k && keys[e0 - 1] == k) return;  // the run began earlier
  // the last chunk that begins with k
  int end = chunk + 1;
  for (;;) {
    const int64_t e = (int64_t)(end + lane) * CHUNK;
    const uint64_t m = __ballot(e < N && keys[e < N ? e : 0] == k);
    const int run = m == ~0ull ? 64 : __builtin_ctzll(~m);
    end += run;
    if (run < 64) break;
  }
  const int64_t c = (int64_t)blockIdx.y * 64 * VEC + lane * VEC;
  float sum[VEC];
#pragma unroll
  for (int x = 0; x < VEC; ++x) sum[x] = 0.0f;
  if (c < D) {
    if (wave == 0) loadv<F32, VEC>((const uint8_t*)(tail + (int64_t)chunk * D + c), sum);
    for (int h = chunk + 1 + wave; h < end; h += 8) {
      float v[VEC];
      loadv<F32, VEC>((const uint8_t*)(head + (int64_t)h * D + c), v);
#pragma unroll
      for (int x = 0; x < VEC; ++x) sum[x] += v[x];
    }
  }
#pragma unroll
  for (int x = 0; x < VEC; ++x) part[wave][lane * VEC + x] = sum[x];
  __syncthreads();
  if (wave != 0 || c >= D) return;
#pragma unroll
  for (int w = 1; w < 8; ++w)
#pragma unroll
    for (int x = 0; x < VEC; ++x) sum[x] += part[w][lane * VEC + x];
  put_row<OT, VEC>(out + ((int64_t)k * D + c) * OB, sum, factor, accumulate);
}

__global__ __launch_bounds__(256) void embedding_zero_kernel(ti_u32x4* __restrict__ p, int64_t n16,
                                                             uint16_t* __restrict__ rest, int nr) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n16; i += (int64_t)gridDim.x * 256)
    p[i] = ti_u32x4{0u, 0u, 0u, 0u};
  if (blockIdx.x == 0 && (int)threadIdx.x < nr) rest[threadIdx.x] = 0;
}

size_t align256(size_t b) { return (b + 255) & ~(size_t)255; }

struct EmbedPlan {
  int passes, per, blocks;
  int64_t chunks;
  size_t hist, keys[2], pos[2], head, tail, total;
};

EmbedPlan embed_plan(int64_t N, int64_t V, int64_t D) {
  EmbedPlan p{};
  int bits = 1;
  while (bits < 33 && ((int64_t)1 << bits) <= V) ++bits;  // keys 0 .. V
  p.passes = (bits + DIGIT - 1) / DIGIT;
  // 2048 entries a block, more when that makes over 128 blocks; 256 divide it
  p.per = (int)std::max<int64_t>(2048, ((N + BLOCKS - 1) / BLOCKS + 255) / 256 * 256);
  p.blocks = (int)((N + p.per - 1) / p.per);
  p.chunks = (N + CHUNK - 1) / CHUNK;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t b = at;
    at += align256(bytes);
    return b;
  };
  p.hist = take((size_t)p.blocks * BINS * 4);
  for (int i = 0; i < 2; ++i) p.keys[i] = take((size_t)N * 4), p.pos[i] = take((size_t)N * 4);
  p.head = take((size_t)p.chunks * D * 4);
  p.tail = take((size_t)p.chunks * D * 4);
  p.total = at;
  return p;
}

template <int GT, int OT, int VEC>
int sums(const EmbedPlan& p, const uint8_t* grad, const uint32_t* keys, const uint32_t* pos,
         int64_t N, int64_t V, int64_t D, float factor, int accumulate, uint8_t* ws, uint8_t* out,
         hipStream_t st) {
  float* head = reinterpret_cast<float*>(ws + p.head);
  float* tail = reinterpret_cast<float*>(ws + p.tail);
  const unsigned cols = (unsigned)((D + 64 * VEC - 1) / (64 * VEC));
  hipLaunchKernelGGL((embedding_sum_kernel<GT, OT, VEC>),
                     dim3((unsigned)((p.chunks + 3) / 4), cols), dim3(256), 0, st, grad, keys, pos,
                     (int)N, V, D, factor, accumulate, head, tail, out);
  int rc = check_launch();
  if (rc != NOVAQ_OK || p.chunks < 2) return rc;
  hipLaunchKernelGGL((embedding_join_kernel<OT, VEC>), dim3((unsigned)p.chunks, cols), dim3(512),
                     0, st, keys, (int)N, V, D, factor, accumulate, head, tail, out);
  return check_launch();
}

template <int GT, int OT>
int sums_by_width(const EmbedPlan& p, const void* grad, const uint32_t* keys, const uint32_t* pos,
                  int64_t N, int64_t V, int64_t D, float factor, int accumulate, uint8_t* ws,
                  void* out, hipStream_t st) {
  const uint8_t* g = static_cast<const uint8_t*>(grad);
  uint8_t* o = static_cast<uint8_t*>(out);
  if (D % 8 == 0) return sums<GT, OT, 8>(p, g, keys, pos, N, V, D, factor, accumulate, ws, o, st);
  if (D % 4 == 0) return sums<GT, OT, 4>(p, g, keys, pos, N, V, D, factor, accumulate, ws, o, st);
  return sums<GT, OT, 1>(p, g, keys, pos, N, V, D, factor, accumulate, ws, o, st);
}

}  // namespace

int embedding_launch(const void* ids, int bits, int64_t N, const void* table, int w_dtype,
                     const float* scale, int64_t V, int64_t D, float factor, void* out,
                     int out_dtype, hipStream_t st) {
  switch (w_dtype) {
    case F32: return lookup_to<F32>(out_dtype, ids, bits, N, table, scale, V, D, factor, out, st);
    case F16: return lookup_to<F16>(out_dtype, ids, bits, N, table, scale, V, D, factor, out, st);
    case BF16: return lookup_to<BF16>(out_dtype, ids, bits, N, table, scale, V, D, factor, out, st);
    case E4M3: return lookup_to<E4M3>(out_dtype, ids, bits, N, table, scale, V, D, factor, out, st);
    case E5M2: return lookup_to<E5M2>(out_dtype, ids, bits, N, table, scale, V, D, factor, out, st);
    case E2M1: return lookup_to<E2M1>(out_dtype, ids, bits, N, table, scale, V, D, factor, out, st);
    default: return NOVAQ_EDTYPE;
  }
}

size_t embedding_backward_workspace(int64_t N, int64_t V, int64_t D) {
  return N > 0 ? embed_plan(N, V, D).total : 0;
}

int embedding_backward_launch(const void* grad, int g_dtype, const void* ids, int bits, int64_t N,
                              int64_t V, int64_t D, float factor, int accumulate, void* out,
                              int o_dtype, void* workspace, hipStream_t st) {
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  if (!accumulate) {
    const int64_t bytes = V * D * (o_dtype == F32 ? 4 : 2), n16 = bytes / 16;
    const unsigned blocks = (unsigned)std::min<int64_t>(std::max<int64_t>((n16 + 255) / 256, 1), 8192);
    hipLaunchKernelGGL(embedding_zero_kernel, dim3(blocks), dim3(256), 0, st,
                       static_cast<ti_u32x4*>(out), n16,
                       reinterpret_cast<uint16_t*>(static_cast<uint8_t*>(out) + n16 * 16),
                       (int)(bytes % 16 / 2));
    const int rc = check_launch();
    if (rc != NOVAQ_OK) return rc;
  }
  if (N == 0) return NOVAQ_OK;
  const EmbedPlan p = embed_plan(N, V, D);
  uint32_t* hist = reinterpret_cast<uint32_t*>(ws + p.hist);
  uint32_t* keys[2] = {reinterpret_cast<uint32_t*>(ws + p.keys[0]),
                       reinterpret_cast<uint32_t*>(ws + p.keys[1])};
  uint32_t* pos[2] = {reinterpret_cast<uint32_t*>(ws + p.pos[0]),
                      reinterpret_cast<uint32_t*>(ws + p.pos[1])};
  for (int i = 0; i < p.passes; ++i) {
    const void* raw = i == 0 ? ids : nullptr;
    const int in = i & 1, to = in ^ 1;
    hipLaunchKernelGGL(sort_hist_kernel, dim3(p.blocks), dim3(256), 0, st, keys[in], raw, bits, V,
                       (int)N, p.per, i * DIGIT, hist);
    int rc = check_launch();
    if (rc != NOVAQ_OK) return rc;
    hipLaunchKernelGGL(sort_scatter_kernel, dim3(p.blocks), dim3(256), 0, st, keys[in], pos[in],
                       raw, bits, V, (int)N, p.per, i * DIGIT, hist, keys[to], pos[to]);
    rc = check_launch();
    if (rc != NOVAQ_OK) return rc;
  }
  const uint32_t* k = keys[p.passes & 1];
  const uint32_t* q = pos[p.passes & 1];
#define NOVAQ_SUMS(G, O) \
  return sums_by_width<G, O>(p, grad, k, q, N, V, D, factor, accumulate, ws, out, st)
#define NOVAQ_SUMS_TO(G)                  \
  if (o_dtype == F32) NOVAQ_SUMS(G, F32); \
  if (o_dtype == F16) NOVAQ_SUMS(G, F16); \
  NOVAQ_SUMS(G, BF16)
  if (g_dtype == F32) { NOVAQ_SUMS_TO(F32); }
  if (g_dtype == F16) { NOVAQ_SUMS_TO(F16); }
  NOVAQ_SUMS_TO(BF16);
#undef NOVAQ_SUMS_TO
#undef NOVAQ_SUMS
}

}  // namespace novaq
