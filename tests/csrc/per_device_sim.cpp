// What is done once on each device (per_device.h), with a status that the test sets.
#include <cstdio>

#include "per_device.h"

enum Status { kOk = 0, kFailed = 7 };

int main() {
  static lasp::PerDevice once;
  int calls = 0, bad = 0;
  Status next = kFailed;
  const auto first = [&] { return ++calls, next; };
  const auto expect = [&](Status got, Status status, int made, const char* what) {
    if (got != status || calls != made) ++bad, std::printf("%s: status %d of %d, %d calls of %d\n", what, got, status, calls, made);
  };
  expect(once.once(0, first), kFailed, 1, "a failure is reported");
  expect(once.once(0, first), kFailed, 2, "and tried again");
  next = kOk;
  expect(once.once(0, first), kOk, 3, "until it succeeds");
  next = kFailed;
  expect(once.once(0, first), kOk, 3, "after which it is not made again");
  expect(once.once(1, first), kFailed, 4, "but on another device it is");
  next = kOk;
  expect(once.once(1, first), kOk, 5, "there, too, until it succeeds");
  expect(once.once(63, first), kOk, 6, "the last device that is counted");
  expect(once.once(63, first), kOk, 6, "once");
  expect(once.once(64, first), kOk, 7, "a device beyond those that are counted");
  expect(once.once(64, first), kOk, 8, "is asked each time");
  expect(once.once(-1, first), kOk, 9, "no device, too");
  if (!bad) std::printf("ok\n");
  return bad != 0;
}
