// Host check of the paged cache's addressing (csrc/mq_paged.hpp) against its
// definition, over raw device values of every kind.
#include <climits>
#include <cstdio>
#include <vector>

#include "mq_paged.hpp"

int main() {
  long bad = 0, checks = 0;
  auto need = [&](bool ok) {
    ++checks;
    bad += !ok;
  };
  const int wild[] = {INT_MIN, INT_MIN + 1, -70, -1, 0, 1, 2, 63, 64, 65, 100, 129, 1000, INT_MAX - 1, INT_MAX};
  // whatever cu, lens and prefix hold: rows that exist, slots that the table names
  for (int rows : {0, 1, 64, 100})
    for (int cap : {8, 128, INT_MAX - 7})
      for (int a : wild)
        for (int b : wild)
          for (int x : wild) {
            for (int pre : wild) {
              const mq::PagedSeq s = mq::paged_seq(3, a, b, true, x, pre, rows, cap);
              need(s.start >= 0 && s.n >= 0 && s.start <= rows && s.n <= rows - s.start);
              need(s.len >= 0 && s.len <= cap && s.prefix >= 0 && s.prefix <= s.len);
              if (a >= 0 && a <= b && b <= rows) need(s.start == a && s.n == b - a);
              if (x >= 0 && x <= cap) need(s.len == x);
              if (pre >= 0 && pre <= s.len) need(s.prefix == pre);
            }
            const mq::PagedSeq one = mq::paged_seq(3, a, b, false, x, 0, rows, cap);
            need(one.start == 3 && one.n == (rows > 3 ? 1 : 0));
          }
  // the span's tiles hold every slot that a row of p0 .. p1 sees, each tile once, none past the cache
  for (int tk : {8, 16, 64})
    for (int len : {0, 1, 15, 16, 17, 64, 65, 200})
      for (int prefix : {0, 1, 16, 40, 150})
        for (int window : {0, 1, 5, 16, 33, 190, INT_MAX})
          for (int p0 : {-130, -1, 0, 1, 15, 16, 63, 64, 150, 199})
            for (int n : {1, 2, 16, 70}) {
              const int pre = prefix < len ? prefix : len, p1 = p0 + n - 1;
              const mq::PagedSpan s = mq::paged_span(p0, p1, len, pre, window, tk);
              need(s.pre >= 0 && s.pre <= s.lo && s.lo <= s.hi && s.count() >= 0);
              std::vector<int> seen((len + tk - 1) / tk + 1, 0);
              for (int i = 0; i < s.count(); ++i) {
                const int t = s.tile(i);
                const bool in = t >= 0 && t * tk < len;
                need(in);
                if (in) need(++seen[t] == 1);
              }
              for (int p = p0; p <= p1 && p < len; ++p)
                for (int j = 0; j < len; ++j) {
                  const bool see = (j <= p && (window <= 0 || p - j < window)) || j < pre;
                  need(mq::paged_visible(p, j, len, pre, window) == see);
                  if (see) need(seen[j / tk] == 1);
                }
            }
  for (int j : wild) need(mq::paged_visible(j, -1, 100, 0, 0) == false && mq::paged_visible(j, 100, 100, 100, 0) == false);
  // pages that are none, and slots outside the sequence (the row must not be read there)
  const int32_t row[] = {0, 9, 10, -1, INT_MIN, INT_MAX, 3};
  const int want[] = {0, 9, -1, -1, -1, -1, 3};
  for (int j = 0; j < 7 * 8; ++j) {
    need(mq::paged_page(row, j, 56, 3, 10) == want[j / 8]);
    need(mq::paged_page(row, j, j, 3, 10) == -1);
  }
  for (int j : {INT_MIN, -1, 56, INT_MAX}) need(mq::paged_page(nullptr, j, 56, 3, 10) == -1);
  std::printf("checks %ld bad %ld\n", checks, bad);
  return bad != 0;
}
