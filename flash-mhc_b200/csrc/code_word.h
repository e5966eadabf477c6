// Words of a row of codes that is read at any place (plain C++, so that the host
// compiles it too).
#pragma once

#include <stdint.h>

namespace fmhc {

// The twelve codes from `at` (a multiple of 4, maybe outside the row) of a row of C: by
// `word` where four of them are the row's own, else one by one by `code`; zeros for what
// is not the row's.  What lies between rows may be another's, and is not read.
template <class Word, class Code>
constexpr void code_words(int at, int C, const Word &word, const Code &code, uint32_t (&q)[3]) {
  for (int j = 0; j < 3; ++j) {
    const int a = at + 4 * j;
    q[j] = a >= 0 && a + 4 <= C ? word(a) : 0u;
  }
  const int last = C & ~3;  // the word that ends behind the row, if C is no multiple of 4
  if (last < C && last >= at && last < at + 12) {
    uint32_t w = uint8_t(code(last));
    if (last + 1 < C) w |= uint32_t(uint8_t(code(last + 1))) << 8;
    if (last + 2 < C) w |= uint32_t(uint8_t(code(last + 2))) << 16;
    for (int j = 0; j < 3; ++j)
      if (at + 4 * j == last) q[j] = w;
  }
}

}  // namespace fmhc
