// What a host thread has been told of the devices' counts of failures.
#pragma once

#include <cstdint>

namespace pb {

// The counts on the devices only grow, so each thread learns of each rise by itself,
// whatever other threads have asked.
struct Told {
  static constexpr int kDevices = 64;
  uint32_t seen[kDevices] = {};
  // Whether the count of `device` has changed since this thread last asked (devices past
  // the last place: whether there is any failure at all).
  bool news(int device, uint32_t count) {
    if (device < 0 || device >= kDevices) return count != 0;
    const bool is = count != seen[device];
    seen[device] = count;
    return is;
  }
};

}  // namespace pb
