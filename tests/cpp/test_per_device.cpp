// Two unlike devices keep answers of their own; an answer of 0 is asked for again.
#include <cstdio>

#include "../../rustorch_b200/csrc/rtb_per_device.h"

#define CHECK(x)                                      \
  if (!(x)) {                                         \
    std::printf("line %d: %s\n", __LINE__, #x);       \
    return 1;                                         \
  }

int main() {
  static rtb::PerDevice<4> known;
  int asked = 0;
  auto answer = [&](int n) { return [&asked, n] { ++asked; return n; }; };
  CHECK(known.get(0, 2, answer(37)) == 37);
  CHECK(known.get(1, 2, answer(16)) == 16);
  CHECK(known.get(0, 3, answer(15)) == 15);
  CHECK(asked == 3);
  CHECK(known.get(0, 2, answer(1)) == 37 && known.get(1, 2, answer(1)) == 16 && asked == 3);
  CHECK(known.get(2, 0, answer(0)) == 0 && known.get(2, 0, answer(5)) == 5 && asked == 5);
  CHECK(known.get(900, 0, answer(7)) == 7 && known.get(900, 0, answer(8)) == 8 && asked == 7);
  std::printf("fine\n");
  return 0;
}
