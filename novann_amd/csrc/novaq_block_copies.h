// What a tile of the block products (block_gemm.h) copies of its operands: the bytes that
// its buffer descriptors allow and the offsets of its lanes.  Plain C++ (no HIP types) so
// that a host compiler can build it on its own; under hipcc these are the device functions
// that the kernel runs.
//
// A descriptor allows a copy that ends within its bytes and gives zeros for one behind them,
// so these have to end where the operand does and never wrap.  All in 32 bits: a tile has at
// most 256 rows of 4 MiB.
#ifndef NOVAQ_BLOCK_COPIES_H
#define NOVAQ_BLOCK_COPIES_H

#include <stdint.h>

#ifdef __HIPCC__
#define NOVAQ_COPIES_HD __host__ __device__
#else
#define NOVAQ_COPIES_HD
#endif

namespace novaq {
namespace block_detail {

// Bytes of the `tile` rows from `first` on that an operand of `rows` rows of ld bytes has.
NOVAQ_COPIES_HD inline uint32_t code_bytes(int64_t rows, int64_t first, int tile, int64_t ld) {
  const int left = (int)rows - (int)first;
  return (uint32_t)(left < tile ? left : tile) * (uint32_t)ld;
}

// How many of them are left from block kb on, where the operand's blocks end at kb1.
NOVAQ_COPIES_HD inline uint32_t codes_left(uint32_t bytes, int kb, int kb1) {
  return kb < kb1 ? bytes - (uint32_t)kb * 128u : 0u;
}

// The offset from the tile's first row of the first 16 bytes that thread tid copies; the
// rows of its next ones follow at a fixed step.
NOVAQ_COPIES_HD inline uint32_t code_offset(int64_t ld, int tid) {
  const int r = tid / 8, c = (tid % 8) ^ ((r >> 1) & 7);
  return (uint32_t)r * (uint32_t)ld + c * 16;
}

// The exponents of 64 rows from `first` on (a row of lde bytes for 2^shift of them): where
// they begin, the bytes that the operand has (none where all rows are past its last), and
// the offset of a lane's row.
struct ExponentSet {
  int64_t from;
  int bytes;
  uint32_t offset;
};
NOVAQ_COPIES_HD inline ExponentSet exponent_set(int64_t rows, int64_t lde, int shift, int first,
                                                int lane) {
  const int row = first >> shift, left = ((int)(rows - 1) >> shift) + 1 - row;
  const int some = left < 64 ? left : 64;
  return ExponentSet{row * lde, (some > 0 ? some : 0) * (int)lde,
                     (uint32_t)(((first + lane) >> shift) - row) * (uint32_t)lde};
}

// How many bytes are left of them from block kb on.
NOVAQ_COPIES_HD inline uint32_t exponents_left(int bytes, int kb, int kb1) {
  const int left = bytes - kb;
  return kb < kb1 && left > 0 ? (uint32_t)left : 0u;
}

}  // namespace block_detail
}  // namespace novaq

#endif  // NOVAQ_BLOCK_COPIES_H
