// Host check of the rows that a block of slots concerns (csrc/mq_paged.hpp)
// against the mask's definition, and at sizes whose products pass 32 bits.
#include <climits>
#include <cstdio>
#include <initializer_list>

#include "mq_paged.hpp"

int main() {
  long bad = 0, checks = 0;
  auto need = [&](bool ok) {
    ++checks;
    bad += !ok;
  };
  // every row that sees a slot of the block is in the range, none outside the chunk
  for (int len : {0, 1, 15, 16, 17, 64, 200})
    for (int n : {0, 1, 2, 16, 70, 250})   // also more tokens than slots
      for (int prefix : {0, 1, 16, 40, 150, 200})
        for (int window : {0, 1, 5, 33, 190, INT_MAX})
          for (int g : {1, 7})
            for (int j0 = 0; j0 < 320; j0 += 16) {
              const mq::PagedSeq s = {0, n, len, prefix < len ? prefix : len};
              const mq::PagedRange r = mq::paged_rows(j0, 16, s, window, g);
              need(r.begin >= 0 && r.begin <= r.end && r.end <= n * g && r.begin % g == 0 && r.end % g == 0);
              if (j0 >= len) need(r.begin == r.end);
              for (int i = 0; i < n; ++i)
                for (int j = j0; j < j0 + 16; ++j)
                  if (mq::paged_visible(len - n + i, j, len, s.prefix, window)) need(i * g >= r.begin && i * g < r.end);
            }
  // short sequences in tables of up to 2^31 slots: nothing past the sequence, whatever the group
  for (int g : {1, 3, 16, 128, 1024, 65536})
    for (int n : {0, 1, 4, 300})
      for (int len : {1, 300, 5000})
        for (int window : {0, 1, INT_MAX})
          for (int64_t j = 0; j < INT_MAX - 256; j = j < 8192 ? j + 256 : j + (INT_MAX / 777 & ~255)) {
            const mq::PagedSeq s = {0, n, len, 0};
            const mq::PagedRange r = mq::paged_rows((int)j, 256, s, window, g);
            need(r.begin >= 0 && r.begin <= r.end && (int64_t)r.end <= (int64_t)n * g);
            if (j >= len) need(r.begin == r.end);
          }
  // as many rows as there may be, at the far end of as long a sequence as there may be
  for (int g : {1, 7, 65535}) {
    const int n = INT_MAX / g, len = INT_MAX - 7;
    for (int window : {0, 1, 1000, INT_MAX})
      for (int j0 : {0, 256, (len - n) / 256 * 256, (len - 1) / 256 * 256}) {
        const mq::PagedSeq s = {0, n, len, 0};
        const mq::PagedRange r = mq::paged_rows(j0, 256, s, window, g);
        need(r.begin >= 0 && r.begin <= r.end && r.end <= n * g);
        if (window == 0) need(r.end == n * g);
      }
  }
  std::printf("checks %ld bad %ld\n", checks, bad);
  return bad != 0;
}
