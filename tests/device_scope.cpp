// Two GPUs that only a counter knows: what DeviceScope asks of the runtime.
#include "device_scope.hpp"

#include <cstdio>

static int current = 0, sets = 0;
extern "C" hipError_t hipGetDevice(int *d) {
  *d = current;
  return hipSuccess;
}
extern "C" hipError_t hipSetDevice(int d) {
  current = d;
  ++sets;
  return hipSuccess;
}

static bool call(int device, bool fail) {
  const vsk::DeviceScope scope(device);
  if (fail) throw 1;
  return current == device;
}

int main() {
  bool ok = call(1, false) && current == 0 && sets == 2;
  current = 1;
  ok = ok && call(1, false) && current == 1 && sets == 2;  // nothing to change
  try {
    call(0, true);
    ok = false;
  } catch (int) {
  }
  ok = ok && current == 1;
  std::puts(ok ? "device scope ok" : "failed");
  return ok ? 0 : 1;
}
