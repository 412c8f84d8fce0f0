// Test-only: the checks of a shared error word (csrc/error_word.cuh) on words of the test's own.  Not part of the product library.
#include "../ateniaengine_b200/csrc/error_word.cuh"

extern "C" int probe_take(void* word, void* taken, void* stream, int* code, int* site) {
  static std::mutex mu;
  atenia::DeviceError e{};
  const int rc = atenia::take_device_error(static_cast<atenia::DeviceError*>(word), static_cast<atenia::DeviceError*>(taken), mu,
                                           static_cast<cudaStream_t>(stream), &e);
  *code = e.code, *site = e.site;
  return rc;
}
