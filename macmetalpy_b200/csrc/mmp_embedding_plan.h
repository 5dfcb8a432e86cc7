// Which rows' zeros each kernel of mmp_embedding_grad writes (more tokens than
// its one launch takes).  Host arithmetic alone, so that it can be checked on
// a host without a GPU.
#pragma once

#include <stdint.h>

namespace mmp {

// Rows [0, first): beside the sort.  [first, second): beside the sums.  From
// `second` on: beside the joining of runs.  The last two read the bitmap of
// the rows that have tokens, a warp `unit` rows at a time out of one 32-bit
// word, so both start at a multiple of 32 (or at the table's end): a unit that
// began elsewhere could reach into the next word, whose rows would pass for
// rows without tokens.
struct EmbZeroPlan {
  unsigned first, second, unit;
};

// `rows` of `row` bytes; `beside_sort`: whether the sort's kernel writes some.
inline EmbZeroPlan emb_zero_plan(int64_t rows, int64_t row, bool beside_sort) {
  EmbZeroPlan p = {0, (unsigned)rows, 32};
  // the sort takes some 10 us: as many zeros beside it as are written in that
  // time.  With 16, 32 and 48 MB: 16384 tokens, 50257 x 2048 float16 69.0, 67.9
  // and 69.9 us; 50257 x 768 float16 39.8, 40.3, 42.3; 8192 tokens, 100000 x 300
  // float32 37.8, 38.6, 40.3; 4096 tokens, 32000 x 4096 float16 68.5, 65.3, 67.6
  const int64_t early = (int64_t)32 << 20;
  if (beside_sort) p.first = (unsigned)(rows * row < early ? rows : early / row / 32 * 32);
  // 24 MB are left for the joining kernel, which waits for memory some 6 us
  // and moves next to nothing (12 and 48 MB are within 2 % at those sizes)
  const int64_t late = ((int64_t)24 << 20) / row;
  if (rows - p.first > 2 * late) p.second = (unsigned)((rows - late) / 32 * 32);
  // 8 KB of rows a warp at a time
  while (p.unit > 1 && p.unit * row > 8192) p.unit /= 2;
  return p;
}

}  // namespace mmp
