// Two neighbours of a row of 16-bit elements as one word, read without a byte
// from outside the row.
#pragma once

#include <cstdint>

namespace pcb {
namespace loss {

// The words that hold elements 2j and 2j + 1 of a row of `cols` elements.  An
// `odd` row starts on an odd multiple of two bytes: its 4-byte words begin at odd
// elements, and a pair lies in two of them.  A word that reaches beyond the row (to
// what stands before its first or behind its last element) is read as the one
// element of it that is the row's.
//
// Row: pair(i), the word of elements i and i + 1, 4-byte aligned; half(i), element i.
struct WordParts {
  uint32_t a, b;
};
template <typename Row>
__host__ __device__ inline WordParts load_word_parts(const Row& row, bool odd, int j, int cols) {
  const int i = 2 * j;
  if (!odd) return WordParts{i + 1 < cols ? row.pair(i) : (uint32_t)row.half(i), 0};
  WordParts w;
  w.a = j > 0 ? row.pair(i - 1) : (uint32_t)row.half(0) << 16;
  w.b = i + 2 < cols ? row.pair(i + 1) : i + 1 < cols ? (uint32_t)row.half(i + 1) : 0u;
  return w;
}
// Element 2j in the low half, 2j + 1 in the high one (0 beyond the row).
__host__ __device__ inline uint32_t join_word_parts(const WordParts& w, bool odd) {
  return odd ? w.a >> 16 | w.b << 16 : w.a;
}

}  // namespace loss
}  // namespace pcb
