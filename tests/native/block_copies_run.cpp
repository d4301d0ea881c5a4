// Test helper: the copies of every tiling of the block products (novaq_block_copies.h, the
// loop of BlockGemm::run) over seeded sizes.  Each copy that its descriptor allows has to lie
// in the operand, one that it refuses to start behind the descriptor's end, and the allowed
// ones have to bring every byte of the tile's rows and every exponent that they are multiplied
// with.  Prints "ok <cases> <copies refused in 64-row sets past an operand>", or the first
// case that fails.  Built with g++ by tests/test_block_copies.py.
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "../../novann_amd/csrc/novaq_block_copies.h"

using namespace novaq::block_detail;

namespace {

struct Tiling {
  int edge, threads, groups;
};
const Tiling tilings[] = {{256, 256, 1}, {128, 256, 1}, {128, 256, 2}, {64, 128, 1}, {64, 128, 2},
                          {64, 128, 4}};
long past = 0;

#define CHECK(c)                                                                              \
  if (!(c)) {                                                                                 \
    std::printf("%s: edge %d threads %d rows %ld ld %ld shift %d first %ld kb %d of %d..%d\n", \
                #c, t.edge, t.threads, (long)rows, (long)ld, shift, (long)m0, kb, kb0, kb1);  \
    return false;                                                                             \
  }

// One group of waves: blocks kb0 to kb1 of one operand's tile, `rounds` of them gone through
// and two stages (the next four blocks' exponents) copied past them.
bool group(const Tiling& t, int64_t rows, int64_t ld, int64_t lde, int shift, int64_t m0, int kb0,
           int kb1, int rounds, bool every) {
  int kb = kb0;
  const uint32_t bytes = code_bytes(rows, m0, t.edge, ld);
  const int64_t size = rows * ld, left = rows - m0 < t.edge ? rows - m0 : t.edge;
  CHECK(left > 0 && (int64_t)bytes == left * ld && bytes < (1u << 31));
  const int step = t.threads / 8, loads = t.edge * 8 / t.threads;
  for (kb = kb0; kb < kb0 + rounds + 2; ++kb) {
    const uint32_t allowed = codes_left(bytes, kb, kb1);
    const int64_t base = m0 * ld + (int64_t)kb * 128;
    CHECK(allowed == 0 || base + allowed == (m0 + left) * ld);
    std::vector<char> seen(every ? left * 8 : 0, 0);
    for (int i = 0; i < loads; ++i)
      for (int tid = 0; tid < t.threads; ++tid) {
        const uint64_t off = (uint64_t)code_offset(ld, tid) + (uint64_t)(i * step) * (uint64_t)ld;
        CHECK(off < (1ull << 32));
        if (off + 16 <= allowed) {
          CHECK(base + (int64_t)off >= 0 && base + (int64_t)off + 16 <= size);
          if (every) seen[(i * step + tid / 8) * 8 + (off % ld) / 16] = 1;
        } else {
          CHECK(off >= allowed);
        }
      }
    if (every && kb < kb1)
      for (char c : seen) CHECK(c);
  }
  const int64_t erows = ((rows - 1) >> shift) + 1, esize = erows * lde;
  for (int r = 0; r < t.edge; r += 64)
    for (kb = kb0; kb < kb0 + rounds + 4; kb += 4)
      for (int lane = 0; lane < 64; ++lane) {
        const ExponentSet s = exponent_set(rows, lde, shift, (int)m0 + r, lane);
        const uint32_t allowed = exponents_left(s.bytes, kb, kb1);
        CHECK(s.bytes >= 0 && (allowed == 0 || s.from + kb + (int64_t)allowed <= esize));
        const bool in = (uint64_t)s.offset + 4 <= allowed;
        if (in) CHECK(s.from + kb + (int64_t)s.offset + 4 <= esize);
        // (a row that is multiplied has its exponents)
        if (m0 + r + lane < rows && kb < kb1) CHECK(in);
        past += s.bytes == 0 && kb > 0;
      }
  return true;
}

}  // namespace

int main(int argc, char** argv) {
  std::mt19937 rng(7);
  auto below = [&](int n) { return (int)(rng() % (unsigned)n); };
  const int cases = argc > 1 ? std::atoi(argv[1]) : 1000;
  for (int c = 0; c < cases; ++c) {
    const Tiling& t = tilings[below(6)];
    const int kind = below(5);
    // (the last ones: as long as rows may be, 256 of them next to 2^30 bytes)
    const int64_t rows = kind == 0 ? 1 + below(3) : kind == 1 ? 1 + below(130) : 1 + below(5000);
    const int wide = below(5);
    const int64_t K = wide == 0 ? 1 + below(128) : wide == 4 && c % 8 == 0 ? (1 << 22) - below(600)
                                                                         : 1 + below(6000);
    const int blocks = (int)((K + 127) / 128), shift = below(2) * 7;
    const int64_t ld = blocks * 128, lde = (blocks + 3) / 4 * 4;
    const int64_t m0 = (int64_t)below((int)((rows + t.edge - 1) / t.edge)) * t.edge;
    // the blocks over workgroups (parts of fours), then over groups of waves, as the kernel does
    int splits = t.edge == 64 && t.groups == 2 ? 1 << below(4) : 1;
    const int per = splits > 1 ? ((blocks + splits - 1) / splits + 3) / 4 * 4 : blocks;
    splits = (blocks + per - 1) / per;
    const int first = below(splits) * per, last = first + per < blocks ? first + per : blocks;
    for (int g = 0; g < t.groups; ++g) {
      int kb0 = first, kb1 = last, rounds = last - first;
      if (t.groups > 1) {
        const int part = ((last - first + t.groups - 1) / t.groups + 3) / 4 * 4;
        const int end = (last + 3) / 4 * 4;
        kb0 = first + g * part < end ? first + g * part : end;
        kb1 = kb0 + part < last ? kb0 + part : last;
        rounds = part < last - first ? part : last - first;
      }
      if (rounds > 24) {  // the first and the last ones
        if (!group(t, rows, ld, lde, shift, m0, kb0, kb1, 6, false)) return 1;
        kb0 += (rounds - 6) / 4 * 4, rounds = 6 + rounds % 4;
      }
      if (!group(t, rows, ld, lde, shift, m0, kb0, kb1, rounds, blocks <= 8)) return 1;
    }
  }
  std::printf("ok %d %ld\n", cases, past);
  return 0;
}
