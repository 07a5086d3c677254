// device_cache.h -- counts that are asked for once per device and key (the
// CTAs of a kernel that an SM keeps resident).  Host code only.
#pragma once

#include <map>
#include <mutex>
#include <utility>

namespace trs {

template <class Key>
class DeviceCache {
 public:
  // The count kept for (device, key), else query()'s.  A query that fails (below
  // 1) counts as 1 this time and is asked again the next.
  template <class Query>
  int get(int device, const Key& key, Query query) {
    std::lock_guard<std::mutex> lock(mu_);
    const auto at = std::make_pair(device, key);
    const auto it = kept_.find(at);
    if (it != kept_.end()) return it->second;
    const int n = query();
    if (n < 1) return 1;
    return kept_[at] = n;
  }

 private:
  std::mutex mu_;
  std::map<std::pair<int, Key>, int> kept_;
};

}  // namespace trs
