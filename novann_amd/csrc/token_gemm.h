// Matrix products of 16-bit operands (bf16 or f16) with fp32 sums for the
// vocabulary loss:
//
//   C[M, N] = sum over k of A(m, k) * B(n, k)
//
// Each operand lies either K-contiguous (element (r, k) at r * ld + k) or
// K-strided (at k * ld + r), ld a multiple of 8 elements and 16-byte aligned.
// Tiles go from memory straight into LDS (buffer_load ... lds, 16 bytes a
// lane), two stages of 64 K in turn; a K-contiguous tile is read into MFMA
// fragments with 16-byte reads, a K-strided one with gfx950's transposing
// read (ds_read_b64_tr_b16; its lane order is in TokenTile::read), so no operand
// needs a transposed copy.  What lies past a matrix's last row reads as zeros
// through the buffer descriptor, whose base moves with the K block, so no
// offset outgrows 32 bits however long an operand is.  A K-contiguous operand's
// rows are whole multiples of 64 K (the callers keep padded copies); K-strided
// rows past K read as zeros; their columns past the matrix read what follows
// them and go into sums that are not stored.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "novaq_convert.h"
#include "novaq_internal.h"

namespace novaq {
namespace {

typedef float tg_f32x16 __attribute__((ext_vector_type(16)));
typedef float tg_f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t tg_u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t tg_u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 tg_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 tg_f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 tg_bf16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) tg_bf16x4 tg_lds_bf16x4;
typedef __attribute__((address_space(3))) void tg_lds_void;

// MFMAs on fragments held as raw words (CT: BF16 or F16): 32 x 32 x 16, and 16 x
// 16 x 32, which moves half as many accumulators an operation.
template <int CT>
__device__ __forceinline__ tg_f32x16 tg_mfma(const tg_u32x4& a, const tg_u32x4& b,
                                             const tg_f32x16& c) {
  if constexpr (CT == BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(tg_bf16x8, a),
                                                   __builtin_bit_cast(tg_bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(tg_f16x8, a),
                                                  __builtin_bit_cast(tg_f16x8, b), c, 0, 0, 0);
}
template <int CT>
__device__ __forceinline__ tg_f32x4 tg_mfma(const tg_u32x4& a, const tg_u32x4& b,
                                            const tg_f32x4& c) {
  if constexpr (CT == BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(tg_bf16x8, a),
                                                   __builtin_bit_cast(tg_bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(tg_f16x8, a),
                                                  __builtin_bit_cast(tg_f16x8, b), c, 0, 0, 0);
}

// fp32 -> the compute type's 16-bit code, nearest even.
template <int CT>
__device__ __forceinline__ uint32_t tg_pack2(float lo, float hi) {
  if constexpr (CT == BF16) {
    return pack_bf16x2(f2u(lo), f2u(hi));
  } else {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    const f16x2 h = {(_Float16)lo, (_Float16)hi};
    return __builtin_bit_cast(uint32_t, h);
  }
}

// 16 bytes a lane from a buffer (descriptor rs, byte offset voff) straight into
// LDS at lds + 16 * lane, lds the same in all lanes.  In assembly because the
// compiler otherwise waits for every copy in flight before each transposing LDS
// read (grad_W's product of 4096 x 4096 x 16384: 546 us so, 447 with this).  A copy
// has no vector output; m0 (its LDS address) is put back; what reads LDS waits for
// it by vmcnt and a barrier.  NT: past the caches, for what is read once.
template <bool NT = false>
__device__ __forceinline__ void tg_copy16(const tg_u32x4& rs, uint32_t voff, uint8_t* lds) {
  const uint32_t at = (uint32_t)(uintptr_t)(tg_lds_void*)lds;
  uint32_t kept;
#define NOVAQ_COPY16(MORE)                                    \
  asm volatile(                                               \
      "s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\t"   \
      "buffer_load_dwordx4 %2, %3, 0 offen" MORE              \
      " lds\n\ts_mov_b32 m0, %0"                              \
      : "=&s"(kept)                                           \
      : "s"(at), "v"(voff), "s"(rs)                           \
      : "memory")
  if constexpr (NT) NOVAQ_COPY16(" nt");
  else NOVAQ_COPY16("");
#undef NOVAQ_COPY16
}

// One operand of a product: rows (M or N) of K elements.
struct TokenOp {
  const uint16_t* p;
  int64_t rows;  // M (or N)
  int64_t ld;    // elements between rows (K-contiguous) or between K (K-strided)
};

constexpr int TG_KB = 64;  // K of a stage: one 128-byte line of a K-contiguous row

// The LDS tile of one operand: R rows (or columns) of 64 K, 128 R bytes.
//   K-contiguous: row r holds 8 chunks of 16 bytes, chunk c at slot
//     c ^ ((r >> 1) & 7): the 16 rows that one 16-byte read touches at a time
//     fall in distinct banks.
//   K-strided: K row k holds R / 8 chunks, chunk c at slot c ^ (4 (k & 3)) ^
//     (2 (k / 8 & 1)): the K rows k .. k + 3 and k + 8 .. k + 11 that half a
//     wave's transposing read touches lie in distinct 32-byte bank ranges.
template <bool KS, int R, int NTH>
struct TokenTile {
  static constexpr int KB = TG_KB;
  static constexpr int bytes = R * KB * 2;
  static constexpr int loads = R * KB / 8 / NTH;  // 16-byte loads a lane a stage
  static constexpr int cpr = KS ? R / 8 : 8;      // chunks a row
  static_assert(R % 32 == 0 && (R * KB / 8) % NTH == 0 && NTH % cpr == 0, "tile shape");

  // byte offsets of this lane's loads from the tile's base in memory
  struct Src {
    const uint16_t* base;
    int64_t left;   // bytes from base to the operand's end
    uint32_t voff;  // of load 0
    uint32_t step;  // from one load to the next
  };

  __device__ static __forceinline__ Src source(const TokenOp& op, int64_t r0, int64_t K, int tid) {
    Src s;
    // (a load's rows are 16 or more further: the swizzle is the same in all)
    constexpr int step = NTH / cpr;
    static_assert(step % 16 == 0, "swizzle");
    const int r = tid / cpr;
    const int c = (tid % cpr) ^ (KS ? 4 * (r & 3) ^ 2 * ((r >> 3) & 1) : ((r >> 1) & 7));
    s.voff = (uint32_t)r * (uint32_t)(op.ld * 2) + c * 16;
    s.step = step * (uint32_t)(op.ld * 2);
    if constexpr (KS) {
      s.base = op.p + r0;
      s.left = (K * op.ld - r0) * 2;
    } else {
      s.base = op.p + r0 * op.ld;
      s.left = (op.rows - r0) * op.ld * 2;
    }
    return s;
  }

  // The buffer descriptor of stage kb (KB K); with `none` one that gives zeros,
  // without touching memory.
  __device__ static __forceinline__ tg_u32x4 stage_of(const Src& s, const TokenOp& op, int kb,
                                                      bool none) {
    const int64_t at = KS ? (int64_t)kb * KB * op.ld * 2 : (int64_t)kb * 128;
    int64_t left = s.left - at;
    left = none || left < 0 ? 0 : left > 0x7FFFFFFF ? 0x7FFFFFFF : left;
    const uint64_t from = (uint64_t)(reinterpret_cast<const uint8_t*>(s.base) + at);
    return tg_u32x4{(uint32_t)from, (uint32_t)(from >> 32), (uint32_t)left, 0x00020000u};
  }

  // Copy i of a stage to lds (this wave's part).
  __device__ static __forceinline__ void copy(const Src& s, const tg_u32x4& rs, int i,
                                              uint8_t* lds, int wave) {
    tg_copy16(rs, s.voff + i * s.step, lds + (i * NTH + wave * 64) * 16);
  }

  // Fragment of 16 rows (from w0 + 16 i) and 32 K (from 32 s): lane l holds row l %
  // 16, K 8 (l / 16) .. + 7.
  //   K-strided: in each group of 16 lanes lane p names 8 bytes (K row p / 4,
  //     columns 4 (p % 4) .. + 3 of a 4 x 16 block) and receives column p of
  //     the block; the second read is 4 K rows further.
  __device__ static __forceinline__ tg_u32x4 read(const uint8_t* lds, int w0, int i, int s,
                                                  int lane) {
    const int q = lane >> 4;
    if constexpr (KS) {
      const int k = 8 * q + ((lane & 15) >> 2);
      const int byte = ((w0 + i * 16) * 2 ^ ((k & 3) * 64) ^ ((q & 1) * 32)) + (lane & 3) * 8;
      const uint8_t* p = lds + (32 * s + k) * (R * 2) + byte;
      const tg_u32x2 lo = __builtin_bit_cast(
          tg_u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4bf16((tg_lds_bf16x4*)p));
      const tg_u32x2 hi = __builtin_bit_cast(
          tg_u32x2,
          __builtin_amdgcn_ds_read_tr16_b64_v4bf16((tg_lds_bf16x4*)(p + 4 * (R * 2))));
      return tg_u32x4{lo[0], lo[1], hi[0], hi[1]};
    } else {
      const int r = lane & 15;
      return *reinterpret_cast<const tg_u32x4*>(lds + (w0 + i * 16 + r) * 128 +
                                                (((4 * s + q) ^ ((r >> 1) & 7)) << 4));
    }
  }
};

// Spreads a step's R LDS reads over its M MFMAs, reads first: in a burst they
// would hold the matrix cores at each step's start.
template <int R, int M, int I = 0>
__device__ __forceinline__ void tg_mix() {
  if constexpr (I < R) {
    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    if constexpr ((I + 1) * M / R > I * M / R)
      __builtin_amdgcn_sched_group_barrier(0x008, (I + 1) * M / R - I * M / R, 0);
    tg_mix<R, M, I + 1>();
  }
}

// The product of one BM x BN tile by WGM x WGN waves of WM x WN: K blocks kb0
// to kb1 of 64.  acc[i][j]: rows wm + 16 i + 4 (lane / 16) + r, column wn + 16 j +
// lane % 16.  After it returns every wave is done with LDS.
//
// Two stages in LDS: one is copied while the other is multiplied (stages of 32 K,
// four or five of them, were no faster: 460 us and 447).
template <int CT, bool AKS, bool BKS, int WM_, int WN_, int WGN_>
struct TokenGemm {
  static constexpr int WM = WM_, WN = WN_, WGM = 2, WGN = WGN_;
  static constexpr int BM = WGM * WM, BN = WGN * WN, NTH = 64 * WGM * WGN;
  static constexpr int MT = WM / 16, NT = WN / 16;
  using A = TokenTile<AKS, BM, NTH>;
  using B = TokenTile<BKS, BN, NTH>;
  static constexpr int stage = A::bytes + B::bytes;
  // (the epilogue that stores P passes its tile through LDS, rows padded)
  static constexpr int out_bytes = BN * (BM * 2 + 16);
  static constexpr int lds_bytes = 2 * stage > out_bytes ? 2 * stage : out_bytes;
  static constexpr int R = MT * (AKS ? 2 : 1) + NT * (BKS ? 2 : 1);  // LDS reads a step
  // Copies are issued one after another behind the barrier, or spread over the
  // step's MFMAs, which they then do not hold up (loss and gradients of 1000 x 784 x
  // 30001: 276 us and 269; of 8192 x 1024 x 50000: 2970 and 2948).  A large tile with
  // a K-strided operand has no registers left for it (two spilled; the gradients of
  // a 16384-class piece of 4096 x 4096: 870 us spread, 858 not).
  static constexpr bool spread = (!AKS && !BKS) || MT * NT <= 16;
  typedef tg_f32x4 Acc[MT][NT];

  struct Frags {
    tg_u32x4 a[MT];
    tg_u32x4 b[NT];
  };

  __device__ static __forceinline__ void run(Acc& acc, const TokenOp& oa, const TokenOp& ob,
                                             int64_t m0, int64_t n0, int64_t K, int kb0, int kb1,
                                             uint8_t* lds) {
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = (wave % WGM) * WM, wn = (wave / WGM) * WN;
    const typename A::Src sa = A::source(oa, m0, K, tid);
    const typename B::Src sb = B::source(ob, n0, K, tid);
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[i][j][r] = 0.0f;

    tg_u32x4 ra, rb;  // the descriptors of the stage that is copied next
    auto aim = [&](int kb) {
      ra = A::stage_of(sa, oa, kb, kb >= kb1);
      rb = B::stage_of(sb, ob, kb, kb >= kb1);
    };
    auto copy = [&](int i, int slot) {
      uint8_t* at = lds + slot * stage;
      if (i < A::loads) A::copy(sa, ra, i, at, wave);
      else B::copy(sb, rb, i - A::loads, at + A::bytes, wave);
    };
    auto read = [&](Frags& f, int slot, const int s) {
      const uint8_t* at = lds + slot * stage;
#pragma unroll
      for (int i = 0; i < MT; ++i) f.a[i] = A::read(at, wm, i, s, lane);
#pragma unroll
      for (int j = 0; j < NT; ++j) f.b[j] = B::read(at + A::bytes, wn, j, s, lane);
    };
    auto multiply = [&](const Frags& f) {
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = tg_mfma<CT>(f.a[i], f.b[j], acc[i][j]);
    };
    // Stage kb in two steps of 32 K, each step's fragments read while the one before
    // is multiplied.  Before step 1: this wave's reads of stage kb and its copies of
    // stage kb + 1 are done (counters), and after the barrier every wave's, so the
    // copy of stage kb + 2 may overwrite kb's slot, and step 0 of kb + 1 be read.
    // Copies are issued past the end too (of zeros), so that the counters are the
    // same in every stage.
    if (kb0 >= kb1) return;
    constexpr int L = A::loads + B::loads, M = MT * NT;
    Frags f[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      aim(kb0 + i);
#pragma unroll
      for (int q = 0; q < L; ++q) copy(q, i);
    }
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(L) : "memory");
    read(f[0], 0, 0);
    int slot = 0;
    for (int kb = kb0; kb < kb1; ++kb, slot ^= 1) {
      read(f[1], slot, 1);
      multiply(f[0]);
      tg_mix<R, M>();
      if constexpr (spread) aim(kb + 2);
      __builtin_amdgcn_sched_barrier(0);
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (spread) {
        // one read an MFMA, then the copies over the rest of the MFMAs
        const uint8_t* at = lds + (slot ^ 1) * stage;
#pragma unroll
        for (int q = 0; q < M; ++q) {
          const int c = q - MT - NT;  // MFMAs past the reads
          if (q < MT) f[0].a[q] = A::read(at, wm, q, 0, lane);
          else if (c < 0) f[0].b[q - MT] = B::read(at + A::bytes, wn, q - MT, 0, lane);
          acc[q / NT][q % NT] = tg_mfma<CT>(f[1].a[q / NT], f[1].b[q % NT], acc[q / NT][q % NT]);
#pragma unroll
          for (int i = 0; i < L; ++i)
            if (c >= 0 && i >= c * L / (M - MT - NT) && i < (c + 1) * L / (M - MT - NT))
              copy(i, slot);
          __builtin_amdgcn_sched_barrier(0);
        }
      } else {
        aim(kb + 2);
#pragma unroll
        for (int i = 0; i < L; ++i) copy(i, slot);
        read(f[0], slot ^ 1, 0);
        multiply(f[1]);
        tg_mix<R, M>();
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  }
};

}  // namespace
}  // namespace novaq
