// Embedding lookup in a table of any stored type, and its gradient by sorted
// tokens.
//
//   out[i]     = dec(W[t[i]]) * (s * factor)
//   grad_W[v] (+)= factor * sum over i with t[i] = v of grad[i]
//
// The lookup moves one row a token and is bound by memory; 8 elements a lane.
//
// The gradient of few tokens is one launch in which each token's first position
// looks for the others (embedding_few_kernel).  For more it sorts the tokens
// (stable, radix digits of 9 bits), so that a row's positions lie together in
// rising order, and sums chunks of 16 (up to 4096 tokens: 4) sorted entries a
// wave.  A token with many positions spans several of these chunks: each then
// leaves its part in the workspace and a last kernel adds a run's parts in order.
// No atomics touch floating-point values: the sums' order depends on the tokens
// alone, and the result is the same bit for bit in every call.  Sums are fp32; the
// factor is applied once to the whole sum.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "novaq_internal.h"
#include "token_io.h"

namespace novaq {
namespace {

// A row per token, 8 elements a thread and four such units a thread, whose ids
// and then codes are all loaded before the first store; a token outside the table
// gives a row of NaN.  32768 tokens of 1024 E4M3 to bf16: 17 us, 67 MB written and
// 19 read at 5.0 TB/s.
template <int ST, int OT, bool VEC>
__global__ __launch_bounds__(256) void embedding_kernel(const void* __restrict__ ids, int bits,
                                                        const uint8_t* __restrict__ table,
                                                        const float* __restrict__ scale,
                                                        int64_t V, int64_t D, float factor,
                                                        int64_t i0, uint32_t units, uint32_t per,
                                                        FastDiv by_per, void* __restrict__ out) {
  constexpr int A = 4;
  const int64_t rb = row_bytes(ST, D);
  const float a = (scale ? *scale : 1.0f) * factor;
  const uint32_t q0 = blockIdx.x * (256 * A) + threadIdx.x;
  int64_t t[A], i[A], c[A];
#pragma unroll
  for (int k = 0; k < A; ++k) {
    const uint32_t q = min(q0 + k * 256, units - 1), r = fdiv(q, by_per);
    i[k] = i0 + r;
    c[k] = (int64_t)(q - r * per) * 8;
    t[k] = token_at(ids, bits, i[k]);
  }
  float v[A][8];
#pragma unroll
  for (int k = 0; k < A; ++k) {
    const bool in = t[k] >= 0 && t[k] < V;
    load8<ST, VEC>(table + (in ? t[k] : 0) * rb, c[k], D, v[k]);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[k][e] = in ? v[k][e] * a : u2f(0x7FC00000u);
  }
#pragma unroll
  for (int k = 0; k < A; ++k)
    if (q0 + k * 256 < units) store8<OT, VEC>(out, i[k] * D + c[k], D - c[k], v[k]);
}

template <int ST, int OT>
int lookup(const void* ids, int bits, int64_t N, const void* table, const float* scale, int64_t V,
           int64_t D, float factor, void* out, hipStream_t st) {
  const int64_t per = (D + 7) / 8, most = (int64_t)1 << 30;  // units a launch
  const uint8_t* t = static_cast<const uint8_t*>(table);
  for (int64_t i0 = 0; i0 < N; i0 += most / per) {
    const uint32_t units = (uint32_t)(std::min(N - i0, most / per) * per);
    const dim3 grid((units + 1023) / 1024);
    if (D % 8 == 0)
      hipLaunchKernelGGL((embedding_kernel<ST, OT, true>), grid, dim3(256), 0, st, ids, bits, t,
                         scale, V, D, factor, i0, units, (uint32_t)per, fast_div((uint32_t)per),
                         out);
    else
      hipLaunchKernelGGL((embedding_kernel<ST, OT, false>), grid, dim3(256), 0, st, ids, bits, t,
                         scale, V, D, factor, i0, units, (uint32_t)per, fast_div((uint32_t)per),
                         out);
    const int rc = check_launch();
    if (rc != NOVAQ_OK) return rc;
  }
  return NOVAQ_OK;
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
// the sort, and the zeros under it

constexpr int DIGIT = 9, BINS = 1 << DIGIT;
constexpr int BATCH = 1024;     // entries of a block's batch: 4 a lane
constexpr int BLOCKS = 128;     // at most, of a pass
// Entries that one workgroup sorts in LDS (4096: 15 us against 21 for the four
// launches of the passes over blocks; 8192: 24 against 21).
constexpr int SMALL = 4096;

// The rows that get no gradient must be zero: the sort's launches, which use few
// workgroups, carry the table's zeros in their other ones (32768 tokens, a table
// of 205 MB: 31 us of sorting and 28 of writing one after the other, 44 together).
struct Zeros {
  uint8_t* p;
  int64_t from, to;  // bytes, multiples of 16 but for the table's end
  bool past;         // past the caches
};

// A table of more than half the 256 MB cache is written past it: what else the
// cache holds is read next (lookup and gradient of 32768 tokens, 205 MB: 104 us
// through it, 100 past it; of 1000 tokens, 94 MB: 26.3 and 29.3).
constexpr int64_t PAST = (int64_t)128 << 20;

template <bool NT>
__device__ __forceinline__ void write_vectors(ti_u32x4* p, int64_t n, int64_t first, int64_t step) {
  for (int64_t i = first; i < n; i += step) vstore<NT>(p + i, ti_u32x4{0u, 0u, 0u, 0u});
}
__device__ __forceinline__ void write_zeros(const Zeros& z, int block, int blocks, int threads) {
  ti_u32x4* p = reinterpret_cast<ti_u32x4*>(z.p + z.from);
  const int64_t n16 = (z.to - z.from) / 16, step = (int64_t)blocks * threads;
  const int64_t first = (int64_t)block * threads + threadIdx.x;
  if (z.past) write_vectors<true>(p, n16, first, step);
  else write_vectors<false>(p, n16, first, step);
  if (block == 0 && (int64_t)threadIdx.x < (z.to - z.from) % 16)
    z.p[z.from + n16 * 16 + threadIdx.x] = 0;
}

__global__ __launch_bounds__(256) void embedding_zero_kernel(Zeros z) {
  write_zeros(z, blockIdx.x, gridDim.x, 256);
}

// The sort's key of position i: the token, or V where it is none of the
// table's (those sort last and are left out).
__device__ __forceinline__ uint32_t token_key(const void* ids, int bits, int64_t i, int64_t V) {
  const int64_t t = token_at(ids, bits, i);
  return t >= 0 && t < V ? (uint32_t)t : (uint32_t)V;
}

// Exclusive prefix sums of 64 lanes' values.
__device__ __forceinline__ uint32_t wave_before(uint32_t v, int lane, uint32_t& total) {
  uint32_t s = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t o = __shfl_up(s, d);
    if (lane >= d) s += o;
  }
  total = __shfl(s, 63);
  return s - v;
}

// Where the wave's 64 entries of digit d go: cnt[d] holds the next place of each
// digit; equal digits are ranked by ballots and the place moved on by the first of
// them (after the reads of this step, before those of the next).
__device__ __forceinline__ uint32_t place(uint32_t* cnt, uint32_t d, bool in, int lane) {
  uint64_t same = __ballot(in);
#pragma unroll
  for (int bit = 0; bit < DIGIT; ++bit) {
    const uint64_t m = __ballot((d >> bit) & 1);
    same &= (d >> bit) & 1 ? m : ~m;
  }
  const uint32_t rank = __popcll(same & ((1ull << lane) - 1));
  uint32_t at = 0;
  if (in) at = cnt[d] + rank;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  if (in && rank == 0) cnt[d] += (uint32_t)__popcll(same);
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  return at;
}

// Up to 1024 PER entries sorted by one workgroup in LDS, all passes; the other
// workgroups write zeros.
template <int PER>
struct SmallSort {
  static constexpr int W = 16, N = 1024 * PER;
  static constexpr size_t lds = (size_t)(2 * N + W * BINS + W) * 4;
};

template <int PER>
__global__ __launch_bounds__(1024) void sort_small_kernel(const void* __restrict__ ids, int bits,
                                                          int64_t V, int N, int passes,
                                                          uint32_t* __restrict__ keys_out,
                                                          uint32_t* __restrict__ pos_out,
                                                          Zeros z) {
  if (blockIdx.x > 0) {
    write_zeros(z, blockIdx.x - 1, gridDim.x - 1, 1024);
    return;
  }
  constexpr int W = SmallSort<PER>::W;
  extern __shared__ uint32_t small_lds[];
  uint32_t* key = small_lds;
  uint32_t* pos = key + SmallSort<PER>::N;
  uint32_t(*cnt)[BINS] = reinterpret_cast<uint32_t(*)[BINS]>(pos + SmallSort<PER>::N);
  uint32_t* sums = &cnt[W][0];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  // wave w holds entries w 64 PER .. : step i's are 64 i + lane of them
  const int e0 = wave * 64 * PER + lane;
  uint32_t k[PER], p[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = e0 + i * 64;
    k[i] = e < N ? token_key(ids, bits, e, V) : 0u;
    p[i] = (uint32_t)e;
  }
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = pass * DIGIT;
    for (int i = tid; i < W * BINS; i += 1024) cnt[0][i] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (e0 + i * 64 < N) atomicAdd(&cnt[wave][(k[i] >> shift) & (BINS - 1)], 1u);
    __syncthreads();
    // digit tid (of the first 8 waves): its entries in all waves, then the digits
    // before it
    uint32_t all = 0, of_wave, at = 0;
    if (tid < BINS) {
#pragma unroll
      for (int w = 0; w < W; ++w) all += cnt[w][tid];
      at = wave_before(all, lane, of_wave);
      if (lane == 0) sums[wave] = of_wave;
    }
    __syncthreads();
    if (tid < BINS) {
      for (int w = 0; w < wave; ++w) at += sums[w];
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const uint32_t c = cnt[w][tid];
        cnt[w][tid] = at;
        at += c;
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const bool in = e0 + i * 64 < N;
      const uint32_t to = place(cnt[wave], (k[i] >> shift) & (BINS - 1), in, lane);
      if (in) key[to] = k[i], pos[to] = p[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (e0 + i * 64 < N) k[i] = key[e0 + i * 64], p[i] = pos[e0 + i * 64];
  }
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (e0 + i * 64 < N) keys_out[e0 + i * 64] = k[i], pos_out[e0 + i * 64] = p[i];
}

// Digit counts of each block's `per` entries: hist[block][digit].
__global__ __launch_bounds__(256) void sort_hist_kernel(const uint32_t* __restrict__ keys,
                                                        const void* __restrict__ ids, int bits,
                                                        int64_t V, int N, int per, int nb,
                                                        int shift, uint32_t* __restrict__ hist,
                                                        Zeros z) {
  if ((int)blockIdx.x >= nb) {
    write_zeros(z, blockIdx.x - nb, gridDim.x - nb, 256);
    return;
  }
  __shared__ uint32_t cnt[BINS];
  for (int d = threadIdx.x; d < BINS; d += 256) cnt[d] = 0;
  __syncthreads();
  const int from = blockIdx.x * per, to = min(N, from + per);
  for (int i0 = from + threadIdx.x; i0 < to; i0 += BATCH) {
    uint32_t k[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int i = min(i0 + 256 * x, to - 1);
      k[x] = ids ? token_key(ids, bits, i, V) : keys[i];
    }
#pragma unroll
    for (int x = 0; x < 4; ++x)
      if (i0 + 256 * x < to) atomicAdd(&cnt[(k[x] >> shift) & (BINS - 1)], 1u);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < BINS; d += 256) hist[blockIdx.x * BINS + d] = cnt[d];
}

// One stable pass: entry i of digit d goes behind all entries of smaller
// digits, those of d in earlier blocks, and those of d before it in its block.
// Each wave takes a contiguous quarter of the block, 64 entries a step.
__global__ __launch_bounds__(256) void sort_scatter_kernel(
    const uint32_t* __restrict__ keys, const uint32_t* __restrict__ pos,
    const void* __restrict__ ids, int bits, int64_t V, int N, int per, int nb, int shift,
    const uint32_t* __restrict__ hist, uint32_t* __restrict__ keys_out,
    uint32_t* __restrict__ pos_out, Zeros z) {
  if ((int)blockIdx.x >= nb) {
    write_zeros(z, blockIdx.x - nb, gridDim.x - nb, 256);
    return;
  }
  __shared__ uint32_t cnt[4][BINS], sums[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int b = blockIdx.x;
  const int quarter = per / 4, from = b * per + wave * quarter, to = min(N, from + quarter);
  auto batch = [&](int i0, uint32_t(&k)[4], uint32_t(&p)[4]) {
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int i = min(i0 + 64 * x + lane, to - 1);
      k[x] = ids ? token_key(ids, bits, i, V) : keys[i];
      p[x] = ids ? (uint32_t)i : pos[i];
    }
  };
  // the waves' own counts
  for (int w = 0; w < 4; ++w) cnt[w][2 * tid] = 0, cnt[w][2 * tid + 1] = 0;
  uint32_t k[4], p[4];
  if (from < to) batch(from, k, p);
  __syncthreads();
  for (int i0 = from; i0 < to; i0 += 256) {
    if (i0 > from) batch(i0, k, p);
#pragma unroll
    for (int x = 0; x < 4; ++x)
      if (i0 + 64 * x + lane < to) atomicAdd(&cnt[wave][(k[x] >> shift) & (BINS - 1)], 1u);
  }
  // digits 2 tid and 2 tid + 1: entries of earlier blocks, and of all
  uint32_t before[2] = {0, 0}, all[2] = {0, 0};
#pragma unroll 8
  for (int i = 0; i < nb; ++i) {
    const uint2 h = reinterpret_cast<const uint2*>(hist + i * BINS)[tid];
    all[0] += h.x, all[1] += h.y;
    before[0] += i < b ? h.x : 0u, before[1] += i < b ? h.y : 0u;
  }
  uint32_t of_wave;
  uint32_t first = wave_before(all[0] + all[1], lane, of_wave);
  if (lane == 0) sums[wave] = of_wave;
  __syncthreads();
  for (int w = 0; w < wave; ++w) first += sums[w];
  uint32_t at[2] = {first + before[0], first + all[0] + before[1]};
#pragma unroll
  for (int w = 0; w < 4; ++w)
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const uint32_t c = cnt[w][2 * tid + x];
      cnt[w][2 * tid + x] = at[x];
      at[x] += c;
    }
  __syncthreads();
  for (int i0 = from; i0 < to; i0 += 256) {
    if (quarter > 256) batch(i0, k, p);  // (a single batch is still in registers)
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const bool in = i0 + 64 * x + lane < to;
      const uint32_t o = place(cnt[wave], (k[x] >> shift) & (BINS - 1), in, lane);
      if (in) keys_out[o] = k[x], pos_out[o] = p[x];
    }
  }
}

// --------------------------------------------------------------------------
// the sums

// VEC elements from p as fp32 (VEC 8: 16-byte loads; 4: one load).
template <int GT, int VEC, bool NT = false>
__device__ __forceinline__ void loadv(const uint8_t* p, float (&v)[VEC]) {
  if constexpr (VEC == 8) {
    load8<GT, true, NT>(p, 0, 8, v);
  } else if constexpr (VEC == 4) {
    if constexpr (GT == F32) {
      const ti_u32x4 a = vload<NT>(reinterpret_cast<const ti_u32x4*>(p));
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = u2f(a[i]);
    } else {
      const ti_u32x2 a = vload<NT>(reinterpret_cast<const ti_u32x2*>(p));
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
template <int GT, int OT, int VEC, int CHUNK>
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
    loadv<GT, VEC, true>(grad + ((int64_t)pos[e] * D + c) * GB, v[i]);
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
// sums are added in the waves' order.  The launch's chunks start at chunk0.
template <int OT, int VEC>
__global__ __launch_bounds__(512) void embedding_join_kernel(
    const uint32_t* __restrict__ keys, int chunk0, int N, int CHUNK, int64_t V, int64_t D,
    float factor, int accumulate, const float* __restrict__ head, const float* __restrict__ tail,
    uint8_t* __restrict__ out) {
  constexpr int OB = OT == F32 ? 4 : 2;
  __shared__ float part[8][64 * VEC];
  const int chunk = chunk0 + (int)blockIdx.x, lane = threadIdx.x & 63;
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
    for (int h = chunk + 1 + wave; h < end; h += 32) {
      float v[4][VEC];  // (all four loaded before the first is added)
#pragma unroll
      for (int y = 0; y < 4; ++y)
        loadv<F32, VEC>((const uint8_t*)(head + (int64_t)min(h + 8 * y, end - 1) * D + c), v[y]);
#pragma unroll
      for (int y = 0; y < 4; ++y)
        if (h + 8 * y < end) {
#pragma unroll
          for (int x = 0; x < VEC; ++x) sum[x] += v[y][x];
        }
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

// --------------------------------------------------------------------------
// few tokens, without a sort

// At most so many tokens, and workgroups for them (each reads all tokens), and a
// table that the caches hold.  The gradient on this path and by the sort: 64 tokens
// of 512, a table of 10000 rows: 5.6 us and 10.8; 512 of 64, 1000 rows: 4.2 and
// 11.8; 512 of 784, 30001 rows: 16.7 and 18.9, all of them one token 30.5 and 22.4
// (its rows then go through one CU).  1000 of 784 would be 21.3 and 20.5, 64 of 4096
// in a table of 2.1 GB 423 and 395.
constexpr int FEW = 512, FEW_WORK = 1024;
static_assert(FEW == 512, "a token a thread");
constexpr int FEW_ROWS = 1024;  // of the table, at most, of a workgroup that writes zeros

// One launch.  The workgroups x < N take position x and 64 VEC columns each: all
// tokens are compared with the position's own, and where it is the token's first
// its positions' rows are summed, every eighth by a wave and the waves' sums in
// order.  The others take rows of the table: they mark those of the tokens and
// write zeros to the rest.
template <int GT, int OT, int VEC>
__global__ __launch_bounds__(512) void embedding_few_kernel(
    const uint8_t* __restrict__ grad, const void* __restrict__ ids, int bits, int N, int64_t V,
    int64_t D, float factor, int accumulate, int rows, FastDiv by_per,
    uint8_t* __restrict__ out) {
  constexpr int GB = GT == F32 ? 4 : 2, OB = OT == F32 ? 4 : 2;
  __shared__ union {
    struct {
      float part[8][64 * VEC];
      uint64_t mask[8];
      uint16_t list[FEW];
    };
    uint32_t marked[FEW_ROWS / 32];
  } sh;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t t = tid < N ? token_at(ids, bits, tid) : -1;
  if ((int)blockIdx.x >= N) {
    const int64_t r0 = ((int64_t)(blockIdx.x - N) * gridDim.y + blockIdx.y) * rows;
    if (r0 >= V) return;
    const int n = (int)min((int64_t)rows, V - r0);
    for (int i = tid; i < FEW_ROWS / 32; i += 512) sh.marked[i] = 0;
    __syncthreads();
    if (t >= r0 && t < r0 + n) atomicOr(&sh.marked[(t - r0) >> 5], 1u << ((t - r0) & 31));
    __syncthreads();
    // words of 16 bytes, or what 4 elements or 1 are
    using W = std::conditional_t<
        VEC == 8 || (VEC == 4 && OB == 4), ti_u32x4,
        std::conditional_t<VEC == 4, ti_u32x2, std::conditional_t<OB == 4, uint32_t, uint16_t>>>;
    const uint32_t per = (uint32_t)(D * OB / (int)sizeof(W)), all = per * (uint32_t)n;
    W* p = reinterpret_cast<W*>(out + r0 * D * OB);
    const W zero = {};
    for (uint32_t i0 = tid; i0 < all; i0 += 4 * 512) {
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const uint32_t i = i0 + 512 * x, r = fdiv(min(i, all - 1), by_per);
        if (i < all && !(sh.marked[r >> 5] >> (r & 31) & 1)) p[i] = zero;
      }
    }
    return;
  }
  const int at = (int)blockIdx.x;
  const int64_t mine = token_at(ids, bits, at);
  if (mine < 0 || mine >= V) return;
  const uint64_t here = __ballot(t == mine);
  if (lane == 0) sh.mask[wave] = here;
  __syncthreads();
  // the positions in rising order
  int count = 0, before = 0;
#pragma unroll
  for (int w = 0; w < 8; ++w) {
    const uint64_t m = sh.mask[w];
    // (one before `at`: that one's workgroup sums the row)
    if (w < at / 64 ? m != 0 : w == at / 64 && (m & ((1ull << (at & 63)) - 1)) != 0) return;
    if (w < wave) before += __popcll(m);
    count += __popcll(m);
  }
  if (t == mine) sh.list[before + __popcll(here & ((1ull << lane) - 1))] = (uint16_t)tid;
  __syncthreads();
  const int64_t c = (int64_t)blockIdx.y * 64 * VEC + lane * VEC;
  float sum[VEC];
#pragma unroll
  for (int x = 0; x < VEC; ++x) sum[x] = 0.0f;
  if (c < D)
    for (int e = wave; e < count; e += 64) {
      float v[8][VEC];  // (all eight loaded before the first is added)
#pragma unroll
      for (int y = 0; y < 8; ++y)
        loadv<GT, VEC, true>(grad + ((int64_t)sh.list[min(e + 8 * y, count - 1)] * D + c) * GB,
                             v[y]);
#pragma unroll
      for (int y = 0; y < 8; ++y)
        if (e + 8 * y < count) {
#pragma unroll
          for (int x = 0; x < VEC; ++x) sum[x] += v[y][x];
        }
    }
  if (count > 1) {
#pragma unroll
    for (int x = 0; x < VEC; ++x) sh.part[wave][lane * VEC + x] = sum[x];
    __syncthreads();
    if (wave == 0)
      for (int w = 1; w < min(8, count); ++w)
#pragma unroll
        for (int x = 0; x < VEC; ++x) sum[x] += sh.part[w][lane * VEC + x];
  }
  if (wave == 0 && c < D)
    put_row<OT, VEC>(out + (mine * D + c) * OB, sum, factor, accumulate);
}

template <int GT, int OT, int VEC>
int few_launch(const uint8_t* grad, const void* ids, int bits, int64_t N, int64_t V, int64_t D,
               float factor, int accumulate, uint8_t* out, hipStream_t st) {
  constexpr int OB = OT == F32 ? 4 : 2;
  constexpr int word = VEC == 8 ? 16 : VEC * OB;
  const int cols = (int)((D + 64 * VEC - 1) / (64 * VEC));
  const int rows = (int)std::min<int64_t>((V + 1023) / 1024, FEW_ROWS);
  const int64_t zeros = accumulate ? 0 : ((V + rows - 1) / rows + cols - 1) / cols;
  hipLaunchKernelGGL((embedding_few_kernel<GT, OT, VEC>), dim3((unsigned)(N + zeros), cols),
                     dim3(512), 0, st, grad, ids, bits, (int)N, V, D, factor, accumulate, rows,
                     fast_div((uint32_t)(D * OB / word)), out);
  return check_launch();
}

size_t align256(size_t b) { return (b + 255) & ~(size_t)255; }

struct EmbedPlan {
  bool few;
  int passes, per, blocks, chunk;
  int64_t chunks;
  size_t hist, keys[2], pos[2], head, tail, total;
};

EmbedPlan embed_plan(int64_t N, int64_t V, int64_t D) {
  EmbedPlan p{};
  const int64_t width = D % 8 == 0 ? 512 : D % 4 == 0 ? 256 : 64;  // columns a workgroup
  p.few = N <= FEW && N * ((D + width - 1) / width) <= FEW_WORK && V * D <= PAST / 4;
  int bits = 1;
  while (bits < 33 && ((int64_t)1 << bits) <= V) ++bits;  // keys 0 .. V
  p.passes = (bits + DIGIT - 1) / DIGIT;
  // whole batches a block, at most 128 blocks
  p.per = (int)(((N + BLOCKS - 1) / BLOCKS + BATCH - 1) / BATCH * BATCH);
  p.blocks = (int)((N + p.per - 1) / p.per);
  p.chunk = N <= SMALL ? 4 : 16;
  p.chunks = (N + p.chunk - 1) / p.chunk;
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
  const dim3 grid((unsigned)((p.chunks + 3) / 4), cols);
  if (p.chunk == 4)
    hipLaunchKernelGGL((embedding_sum_kernel<GT, OT, VEC, 4>), grid, dim3(256), 0, st, grad, keys,
                       pos, (int)N, V, D, factor, accumulate, head, tail, out);
  else
    hipLaunchKernelGGL((embedding_sum_kernel<GT, OT, VEC, 16>), grid, dim3(256), 0, st, grad, keys,
                       pos, (int)N, V, D, factor, accumulate, head, tail, out);
  int rc = check_launch();
  // (a launch's threads stay below 2^32)
  constexpr int64_t most = (int64_t)1 << 22;
  for (int64_t c0 = 0; c0 < p.chunks && p.chunks > 1 && rc == NOVAQ_OK; c0 += most) {
    hipLaunchKernelGGL((embedding_join_kernel<OT, VEC>),
                       dim3((unsigned)std::min(most, p.chunks - c0), cols), dim3(512), 0, st, keys,
                       (int)c0, (int)N, p.chunk, V, D, factor, accumulate, head, tail, out);
    rc = check_launch();
  }
  return rc;
}

template <int GT, int OT>
int sums_by_width(const EmbedPlan& p, const void* grad, const void* ids, int bits,
                  const uint32_t* keys, const uint32_t* pos,
                  int64_t N, int64_t V, int64_t D, float factor, int accumulate, uint8_t* ws,
                  void* out, hipStream_t st) {
  const uint8_t* g = static_cast<const uint8_t*>(grad);
  uint8_t* o = static_cast<uint8_t*>(out);
  if (p.few) {
    if (D % 8 == 0) return few_launch<GT, OT, 8>(g, ids, bits, N, V, D, factor, accumulate, o, st);
    if (D % 4 == 0) return few_launch<GT, OT, 4>(g, ids, bits, N, V, D, factor, accumulate, o, st);
    return few_launch<GT, OT, 1>(g, ids, bits, N, V, D, factor, accumulate, o, st);
  }
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
  const int64_t bytes = accumulate ? 0 : V * D * (o_dtype == F32 ? 4 : 2);
  uint8_t* table = static_cast<uint8_t*>(out);
  // workgroups of `threads` that write n bytes of zeros: 16 vectors a lane, 4096 waves
  auto zero_blocks = [](int64_t n, int threads) {
    return (unsigned)std::min<int64_t>((n + threads * 256 - 1) / (threads * 256),
                                       262144 / threads);
  };
  if (N == 0) {
    if (bytes == 0) return NOVAQ_OK;
    hipLaunchKernelGGL(embedding_zero_kernel, dim3(zero_blocks(bytes, 256)), dim3(256), 0, st,
                       Zeros{table, 0, bytes, bytes > PAST});
    return check_launch();
  }
  const EmbedPlan p = embed_plan(N, V, D);
  uint32_t* hist = reinterpret_cast<uint32_t*>(ws + p.hist);
  uint32_t* keys[2] = {reinterpret_cast<uint32_t*>(ws + p.keys[0]),
                       reinterpret_cast<uint32_t*>(ws + p.keys[1])};
  uint32_t* pos[2] = {reinterpret_cast<uint32_t*>(ws + p.pos[0]),
                      reinterpret_cast<uint32_t*>(ws + p.pos[1])};
  if (!p.few && N <= SMALL) {
    auto small = [&](auto per) -> int {
      constexpr int PER = decltype(per)::value;
      static DeviceFlags raised;
      const int rc = allow_lds(raised, reinterpret_cast<const void*>(&sort_small_kernel<PER>),
                               SmallSort<PER>::lds, SmallSort<PER>::lds);
      if (rc != NOVAQ_OK) return rc;
      hipLaunchKernelGGL(sort_small_kernel<PER>, dim3(1 + zero_blocks(bytes, 1024)), dim3(1024),
                         SmallSort<PER>::lds, st, ids, bits, V, (int)N, p.passes,
                         keys[p.passes & 1], pos[p.passes & 1], Zeros{table, 0, bytes, bytes > PAST});
      return check_launch();
    };
    const int rc = N <= 1024   ? small(std::integral_constant<int, 1>{})
                   : N <= 2048 ? small(std::integral_constant<int, 2>{})
                               : small(std::integral_constant<int, 4>{});
    if (rc != NOVAQ_OK) return rc;
  }
  // the zeros' share of a launch: one part beside the counts, three beside the
  // scatter, which takes about three times as long
  int64_t zero_at = 0;
  int parts = 0;
  auto share = [&](int more) {
    parts += more;
    const int64_t from = zero_at;
    zero_at = parts == 4 * p.passes ? bytes : bytes / (4 * p.passes) * parts / 16 * 16;
    return Zeros{table, from, zero_at, bytes > PAST};
  };
  for (int i = 0; i < p.passes && N > SMALL; ++i) {
    const void* raw = i == 0 ? ids : nullptr;
    const int in = i & 1, to = in ^ 1;
    Zeros z = share(1);
    hipLaunchKernelGGL(sort_hist_kernel, dim3(p.blocks + zero_blocks(z.to - z.from, 256)),
                       dim3(256), 0, st, keys[in], raw, bits, V, (int)N, p.per, p.blocks,
                       i * DIGIT, hist, z);
    int rc = check_launch();
    if (rc != NOVAQ_OK) return rc;
    z = share(3);
    hipLaunchKernelGGL(sort_scatter_kernel, dim3(p.blocks + zero_blocks(z.to - z.from, 256)),
                       dim3(256), 0, st, keys[in], pos[in], raw, bits, V, (int)N, p.per, p.blocks,
                       i * DIGIT, hist, keys[to], pos[to], z);
    rc = check_launch();
    if (rc != NOVAQ_OK) return rc;
  }
  const uint32_t* k = keys[p.passes & 1];
  const uint32_t* q = pos[p.passes & 1];
#define NOVAQ_SUMS(G, O) \
  return sums_by_width<G, O>(p, grad, ids, bits, k, q, N, V, D, factor, accumulate, ws, out, st)
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
