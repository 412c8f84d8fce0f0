// Test-only: one-time preparations (csrc/first_use.cuh) by many threads, compiled with a host compiler.  Not part of the product library.
#include <chrono>
#include <thread>
#include <vector>

#include "../ateniaengine_b200/csrc/first_use.cuh"

// `threads` calls at once, of a preparation that takes `ms`; of them, how many returned success before any preparation had ended
extern "C" int first_use_too_early(int threads, int ms) {
  atenia::FirstUse first;
  std::atomic<int> prepared{0}, early{0}, go{0};
  std::vector<std::thread> pool;
  for (int i = 0; i < threads; ++i)
    pool.emplace_back([&, i] {
      while (!go.load()) std::this_thread::yield();
      std::this_thread::sleep_for(std::chrono::milliseconds(i * ms / threads));  // (some come while the first is at it)
      const int rc = first([&] {
        std::this_thread::sleep_for(std::chrono::milliseconds(ms));
        prepared = 1;
        return 0;
      });
      if (rc != 0 || prepared.load() == 0) early += 1;
    });
  go = 1;
  for (auto& t : pool) t.join();
  return early.load();
}

// Calls of a preparation that fails `failures` times: how often it ran in `calls` calls; `wrong` counts results that were not its own
extern "C" int first_use_runs(int calls, int failures, int* wrong) {
  atenia::FirstUse first;
  int runs = 0;
  *wrong = 0;
  for (int i = 0; i < calls; ++i) {
    const int rc = first([&] { return ++runs <= failures ? 7 : 0; });
    if (rc != (i < failures ? 7 : 0)) *wrong += 1;
  }
  return runs;
}
