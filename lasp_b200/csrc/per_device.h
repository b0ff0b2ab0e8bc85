// What a kernel needs done once on each device, host side, without CUDA: a failure is reported to the call that met it and tried again at the
// next.  (Two threads may do it at once; what is done twice does no harm.)
#pragma once

namespace lasp {

struct PerDevice {
  static constexpr int kDevices = 64;
  bool done[kDevices] = {};
  // first(): a status that is zero where it succeeded
  template <class FIRST>
  auto once(int device, FIRST first) -> decltype(first()) {
    const bool counted = device >= 0 && device < kDevices;
    if (counted && done[device]) return {};
    const auto status = first();
    if (counted && status == decltype(first()){}) done[device] = true;
    return status;
  }
};

}  // namespace lasp
