// The error word that kernels of stateless calls share: one per device, taken by whoever checks first.
#pragma once
#include <mutex>

#include "common.cuh"

namespace atenia {

static __global__ void take_error_kernel(DeviceError* word, DeviceError* taken) {
  taken->code = atomicExch(&word->code, 0);
  taken->site = word->site;
}

// Waits for the stream and takes what is in `word`.  Reading and clearing are one step on the device, so that of two checks one
// returns an error, and what another stream's kernel records meanwhile stays for the next check.  `mu` guards `taken` (the word's
// result in device memory); nobody waits for another one's stream while it is held.
inline int take_device_error(DeviceError* word, DeviceError* taken, std::mutex& mu, cudaStream_t s, DeviceError* out) {
  ATENIA_CUDA_TRY(cudaStreamSynchronize(s));
  std::lock_guard<std::mutex> lk(mu);
  take_error_kernel<<<1, 1, 0, s>>>(word, taken);
  ATENIA_CUDA_TRY(cudaGetLastError());
  ATENIA_CUDA_TRY(cudaMemcpyAsync(out, taken, sizeof *out, cudaMemcpyDeviceToHost, s));
  return (int)cudaStreamSynchronize(s);
}

}  // namespace atenia
