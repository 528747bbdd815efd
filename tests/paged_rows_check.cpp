// rows_meet against a byte map, over small layouts of two tensors in one buffer.
#include "sfk_rows.h"

#include <cstdio>
#include <vector>

using sfk::Rows;

int main() {
  static uint8_t mem[512];
  long checked = 0, meet = 0;
  for (int wa = 1; wa <= 7; wa += 2)
    for (int sa = wa; sa <= wa + 9; sa += 3)
      for (int na = 0; na <= 4; ++na)
        for (int wb = 1; wb <= 6; ++wb)
          for (int sb = wb; sb <= wb + 10; ++sb)
            for (int nb = 0; nb <= 5; ++nb)
              for (int at = 0; at < 130; at += (at > 40 && at < 120) ? 3 : 1) {
                std::vector<char> used(512, 0);
                for (int i = 0; i < na; ++i)
                  for (int x = 0; x < wa; ++x) used[at + i * sa + x] = 1;
                bool want = false;
                for (int j = 0; j < nb; ++j)
                  for (int x = 0; x < wb; ++x) want = want || used[60 + j * sb + x];
                const Rows a{mem + at, sa, wa, na}, b{mem + 60, sb, wb, nb};
                if (sfk::rows_meet(a, b) != want || sfk::rows_meet(b, a) != want) {
                  std::printf("wrong: a at %d stride %d width %d n %d, b stride %d width %d n %d: %d wanted\n", at, sa, wa, na,
                              sb, wb, nb, want);
                  return 1;
                }
                ++checked;
                meet += want;
              }
  // far apart, and more rows than a loop should take
  const Rows far{(void*)0x7f0000000000, 1 << 20, 1 << 10, 1 << 20}, near{(void*)0x1000, 1 << 20, 1 << 10, 1 << 20};
  if (sfk::rows_meet(far, near) || !sfk::rows_meet(far, far) || !sfk::same_rows(far, far)) return 2;
  const Rows between{(void*)(0x7f0000000000 + (1 << 10)), 1 << 20, (1 << 20) - (1 << 10), 1 << 20};
  if (sfk::rows_meet(far, between)) return 3;
  const Rows one{(void*)0x1000, 64, 64, 1}, wide{(void*)0x1000, 128, 64, 1};
  if (!sfk::same_rows(one, wide)) return 4;
  std::printf("ok %ld layouts, %ld meet\n", checked, meet);
  return 0;
}
