// Which dynamic LDS limit each kernel has on each device: the attribute is one
// value of a kernel on a device, and the last one set holds, so it is only ever
// raised.
#pragma once
#include <map>
#include <utility>

namespace wg {

class LdsLimits {
 public:
  // Whether `bytes` are more than the kernel's limit on the device so far.
  bool above(const void *kernel, int dev, int bytes) const {
    const auto it = limits_.find({kernel, dev});
    return it == limits_.end() || bytes > it->second;
  }
  void set(const void *kernel, int dev, int bytes) { limits_[{kernel, dev}] = bytes; }

 private:
  std::map<std::pair<const void *, int>, int> limits_;
};

}  // namespace wg
