// One-time preparation that several host threads may come to at once (a kernel's attributes, a driver function's address).
#pragma once
#include <atomic>

namespace atenia {

class FirstUse {
 public:
  // Runs `prepare` (0: it succeeded) until one run has succeeded, and returns what it returned.  The mark is set behind it: a
  // thread that finds it may rely on what was prepared.  Threads that come meanwhile run it too, so it has to bear that.
  template <typename F>
  int operator()(F&& prepare) {
    if (done_.load(std::memory_order_acquire)) return 0;
    const int rc = prepare();
    if (rc == 0) done_.store(true, std::memory_order_release);
    return rc;
  }

 private:
  std::atomic<bool> done_{false};
};

}  // namespace atenia
