// The vocabulary loss's logits for few tokens (at most 128): the table's codes
// are read once, as stored, and what bounds the kernel is that read.
//
// A workgroup takes 128 or 256 table rows (32 a wave) and all tokens.  Stages of 128
// bytes a row go straight into LDS (whole lines, 16-byte chunks swizzled as in
// TokenTile) beside the tokens' matching K in the order of the MFMA fragments,
// which the call's first kernel lays out: 1 KB a fragment, one coalesced copy.
// A 16-byte chunk of a row holds E codes (8, 16 or 32) and feeds E / 8 MFMAs of
// 16 K: lane half h of chunk pair c takes chunk 2 c + h, and MFMA u its codes 8 u
// .. + 7, so the K of fragment (c, u) are E (2 c + h) + 8 u .. + 7 in both
// operands.  Codes become 16-bit values by the packed converts, exactly.
#pragma once

#include "token_gemm.h"
#include "token_io.h"

namespace novaq {
namespace {

typedef __bf16 ts_bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 ts_f16x2 __attribute__((ext_vector_type(2)));

// 8 codes -> the 4 words of an MFMA fragment.  E4M3 / E5M2: words c0, c1; E2M1:
// c0; 16-bit: the chunk itself (never called).
template <int CT, int WT>
__device__ __forceinline__ tg_u32x4 ts_decode8(uint32_t c0, uint32_t c1) {
  tg_u32x4 o;
#define NOVAQ_CVT(CVT, W, SEL) __builtin_bit_cast(uint32_t, CVT(W, 1.0f, SEL))
  if constexpr (WT == E2M1) {
    if constexpr (CT == BF16) {
      o[0] = NOVAQ_CVT(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4, c0, 0);
      o[1] = NOVAQ_CVT(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4, c0, 1);
      o[2] = NOVAQ_CVT(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4, c0, 2);
      o[3] = NOVAQ_CVT(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4, c0, 3);
    } else {
      o[0] = NOVAQ_CVT(__builtin_amdgcn_cvt_scalef32_pk_f16_fp4, c0, 0);
      o[1] = NOVAQ_CVT(__builtin_amdgcn_cvt_scalef32_pk_f16_fp4, c0, 1);
      o[2] = NOVAQ_CVT(__builtin_amdgcn_cvt_scalef32_pk_f16_fp4, c0, 2);
      o[3] = NOVAQ_CVT(__builtin_amdgcn_cvt_scalef32_pk_f16_fp4, c0, 3);
    }
  } else if constexpr (WT == E4M3) {
    if constexpr (CT == BF16) {
      o[0] = NOVAQ_CVT(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8, c0, false);
      o[1] = NOVAQ_CVT(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8, c0, true);
      o[2] = NOVAQ_CVT(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8, c1, false);
      o[3] = NOVAQ_CVT(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8, c1, true);
    } else {
      o[0] = NOVAQ_CVT(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8, c0, false);
      o[1] = NOVAQ_CVT(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8, c0, true);
      o[2] = NOVAQ_CVT(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8, c1, false);
      o[3] = NOVAQ_CVT(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8, c1, true);
    }
  } else {
    if constexpr (CT == BF16) {
      o[0] = NOVAQ_CVT(__builtin_amdgcn_cvt_scalef32_pk_bf16_bf8, c0, false);
      o[1] = NOVAQ_CVT(__builtin_amdgcn_cvt_scalef32_pk_bf16_bf8, c0, true);
      o[2] = NOVAQ_CVT(__builtin_amdgcn_cvt_scalef32_pk_bf16_bf8, c1, false);
      o[3] = NOVAQ_CVT(__builtin_amdgcn_cvt_scalef32_pk_bf16_bf8, c1, true);
    } else {
      o[0] = NOVAQ_CVT(__builtin_amdgcn_cvt_scalef32_pk_f16_bf8, c0, false);
      o[1] = NOVAQ_CVT(__builtin_amdgcn_cvt_scalef32_pk_f16_bf8, c0, true);
      o[2] = NOVAQ_CVT(__builtin_amdgcn_cvt_scalef32_pk_f16_bf8, c1, false);
      o[3] = NOVAQ_CVT(__builtin_amdgcn_cvt_scalef32_pk_f16_bf8, c1, true);
    }
  }
#undef NOVAQ_CVT
  return o;
}

// Table rows a workgroup, 32 a wave (E codes a chunk, nt tiles of tokens): 128, which
// spreads a small table over more CUs (64 rows of 512 x 10000 E4M3, with gradients:
// 51.8 us, with 256 rows 53.8; of a large table the two are equal), but 256 where
// the tokens' fragments are larger than 128 rows' codes and more rows must share
// them (37 rows of 1024 x 50000 E2M1: 20.1 us a call, with 128 27.5), while two
// stages fit.
constexpr int stream_rows(int E, int nt) { return E * nt > 32 && E * nt < 128 ? 256 : 128; }

template <int CT, int WT, int NT_>
struct TokenStream {
  static constexpr int NT = NT_;                    // tiles of 32 tokens
  static constexpr int E = 128 / dtype_bits(WT);    // codes a chunk
  static constexpr int U = E / 8;                   // MFMAs a chunk
  static constexpr int KS = 8 * E;                  // K a stage (128 bytes a row)
  static constexpr int ROWS = stream_rows(E, NT), NTH = 2 * ROWS;
  static constexpr int w_bytes = ROWS * 128, x_bytes = 4 * U * NT * 1024;
  static constexpr int PASS = NTH * 16;  // bytes that one copy of every lane covers
  static constexpr int WL = w_bytes / PASS, XL = (x_bytes + PASS - 1) / PASS, L = WL + XL;
  static constexpr int stage = w_bytes + XL * PASS;
  // as many stages as leave room for two workgroups a CU, or for one
  static constexpr int ROOM = (2 * stage <= 80 * 1024 ? 80 : 160) * 1024;
  static constexpr int NS = 3 * stage <= ROOM ? 3 : 2;
  static constexpr int lds_bytes = NS * stage;
  static_assert(lds_bytes <= 160 * 1024, "LDS");
  static constexpr int kstages(int64_t D) { return (int)((D + KS - 1) / KS); }

  typedef tg_f32x16 Acc[NT];

  // acc[j]: table rows 32 wave + 8 (r / 4) + 4 (lane / 32) + r % 4 of r0 .., token
  // 32 j + lane % 32.  xf: the tokens' fragments, stage by stage.  Stages are taken
  // from `first` on, around the end: workgroups at the same columns of rows a power
  // of two apart would all read the same few memory channels (one row of 4096 x
  // 131072 E4M3: 94 us all from 0, 78 with every workgroup of an XCD elsewhere).
  __device__ static __forceinline__ void run(Acc& acc, const uint8_t* w, int64_t rows,
                                             int64_t row_bytes, int64_t r0, const uint8_t* xf,
                                             int stages, int first, uint8_t* lds) {
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int chunk = (tid & 7) ^ ((tid >> 4) & 7);  // of row tid / 8 (+ NTH / 8 i)
    const int64_t left = min((int64_t)ROWS, rows - r0) * row_bytes;  // (below 2^30)
    const uint64_t from = (uint64_t)(w + r0 * row_bytes);
    const uint64_t xfrom = (uint64_t)xf;
    const tg_u32x4 xr = {(uint32_t)xfrom, (uint32_t)(xfrom >> 32),
                         (uint32_t)(stages * x_bytes), 0x00020000u};
    const tg_u32x4 wr = {(uint32_t)from, (uint32_t)(from >> 32), (uint32_t)left, 0x00020000u};
    const uint32_t rb = (uint32_t)row_bytes;
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[j][r] = 0.0f;

    // chunks past a row's end and stages past the last one are zeros
    auto issue = [&](int i0, int slot) {
      uint8_t* at = lds + slot * stage + wave * 1024;
      const int s = i0 + first - (i0 + first >= stages ? stages : 0);
      const uint32_t c = (uint32_t)(s * 128 + chunk * 16);
      const uint32_t base = c < rb && i0 < stages ? (uint32_t)(tid >> 3) * rb + c : 0x80000000u;
#pragma unroll
      for (int i = 0; i < WL; ++i)
        tg_copy16<true>(wr, base + i * (NTH / 8) * rb, at + i * PASS);
#pragma unroll
      for (int i = 0; i < XL; ++i) {
        const bool in = i0 < stages && (x_bytes % PASS == 0 || tid * 16 + i * PASS < x_bytes);
        tg_copy16(xr, in ? (uint32_t)(s * x_bytes + tid * 16 + i * PASS) : 0x80000000u,
                  at + w_bytes + i * PASS);
      }
    };
    const int r = lane & 31, h = lane >> 5;
    const int wrow = (wave * 32 + r) * 128;
#pragma unroll
    for (int i = 0; i < NS; ++i) issue(i, i);
    int slot = 0;
    for (int s = 0; s < stages; ++s) {
      asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((NS - 1) * L) : "memory");
      const uint8_t* at = lds + slot * stage;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const tg_u32x4 code = *reinterpret_cast<const tg_u32x4*>(
            at + wrow + (((2 * c + h) ^ ((r >> 1) & 7)) << 4));
#pragma unroll
        for (int u = 0; u < U; ++u) {
          tg_u32x4 a;
          if constexpr (U == 1) a = code;
          else if constexpr (U == 2) a = ts_decode8<CT, WT>(code[2 * u], code[2 * u + 1]);
          else a = ts_decode8<CT, WT>(code[u], 0u);
#pragma unroll
          for (int j = 0; j < NT; ++j)
            acc[j] = tg_mfma<CT>(a,
                                 *reinterpret_cast<const tg_u32x4*>(
                                     at + w_bytes + ((c * U + u) * NT + j) * 1024 + lane * 16),
                                 acc[j]);
        }
      }
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
      issue(s + NS, slot);
      slot = slot + 1 == NS ? 0 : slot + 1;
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
  }
};

}  // namespace
}  // namespace novaq
