// What is set up once for each device, whichever threads call first, in a plain header so that it is tested without a GPU.
#pragma once

#include <map>
#include <mutex>

namespace ei {

template <typename Value>
class PerDevice {
 public:
  // The device's value, made by its first caller while others wait. A set-up that throws is tried again by the next one.
  template <typename Make>
  const Value& get(int device, Make make) {
    const std::lock_guard<std::mutex> lock(mutex_);
    auto found = values_.find(device);
    if (found == values_.end()) found = values_.emplace(device, make()).first;
    return found->second;  // a map's values stay where they are
  }

 private:
  std::mutex mutex_;
  std::map<int, Value> values_;
};

}  // namespace ei
