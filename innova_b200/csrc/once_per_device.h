#pragma once
#include <atomic>
#include <cstdint>

namespace inv {

// What a process asks of each device once, whichever thread comes first. A request that fails (not 0) is made again by the next call, and so is every
// one on a device whose number is outside the word.
class OncePerDevice {
  std::atomic<uint64_t> done_{0};

 public:
  template <typename Request>
  int ask(int device, Request request) {
    const uint64_t bit = device >= 0 && device < 64 ? 1ull << device : 0;
    if (done_.load() & bit) return 0;
    const int error = request();
    if (error == 0) done_.fetch_or(bit);
    return error;
  }
};

}  // namespace inv
