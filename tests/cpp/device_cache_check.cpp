// Host check of tensorrs_b200/csrc/device_cache.h: prints "ok", or the line of
// the first condition that does not hold.
#include <cstdio>
#include <utility>

#include "device_cache.h"

#define CHECK(x) \
  if (!(x)) { std::printf("line %d: %s\n", __LINE__, #x); return 1; }

int main() {
  trs::DeviceCache<std::pair<const void*, int>> c;
  const int k = 0;
  int asked = 0;
  auto give = [&](int n) { return [&asked, n] { ++asked; return n; }; };
  CHECK(c.get(0, {&k, 16}, give(4)) == 4 && asked == 1);
  CHECK(c.get(0, {&k, 16}, give(9)) == 4 && asked == 1);  // kept
  CHECK(c.get(1, {&k, 16}, give(2)) == 2 && asked == 2);  // another device has its own
  CHECK(c.get(0, {&k, 32}, give(3)) == 3 && asked == 3);
  CHECK(c.get(2, {&k, 16}, give(0)) == 1 && asked == 4);  // a failure is 1 this time
  CHECK(c.get(2, {&k, 16}, give(5)) == 5 && asked == 5);  // and asked again
  CHECK(c.get(2, {&k, 16}, give(7)) == 5 && asked == 5);
  std::printf("ok\n");
  return 0;
}
