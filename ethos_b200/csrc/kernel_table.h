// What is asked of the CUDA runtime once per kernel and device: a value per
// (device, kernel), made on first use.  The table has no limit on the kernels:
// one that found no place in it would ask anew at every launch.
#pragma once

#include <mutex>
#include <new>
#include <utility>
#include <vector>

namespace ethos {

template <class V>
class KernelTable {
 public:
  // The value of `fn` on device `dev` into *out; make(V*) fills it the first
  // time.  False, with nothing remembered, when make fails.
  template <class Make>
  bool get(int dev, const void* fn, V* out, Make make) {
    if (dev < 0 || dev >= kDevices) return false;
    std::lock_guard<std::mutex> lock(mu_);
    std::vector<std::pair<const void*, V>>& row = rows_[dev];
    for (const auto& e : row)
      if (e.first == fn) {
        *out = e.second;
        return true;
      }
    if (!make(out)) return false;
    try {  // no exception may pass a C entry point; without memory it is asked again
      row.emplace_back(fn, *out);
    } catch (const std::bad_alloc&) {
    }
    return true;
  }

 private:
  static constexpr int kDevices = 64;
  std::mutex mu_;
  std::vector<std::pair<const void*, V>> rows_[kDevices];
};

}  // namespace ethos
