// A kernel on a device's stream whose one wait runs out: nothing arrives on its
// barrier, so that after about a second it leaves TB200_ERR_TIMEOUT where
// matmul_q8's waits leave it, and returns.
#include "../titania_b200/csrc/runtime.h"

namespace {
__global__ void k_wait_out(int* err) {
  __shared__ uint64_t bar;
  tb::mbar_init(&bar, 1);
  tb::fence_mbar_init();
  tb::mbar_wait(&bar, 0, err);
}
}  // namespace

extern "C" __attribute__((visibility("default"))) int wait_out(tb200_device* d) {
  cudaError_t e = cudaSetDevice(d->ordinal);
  if (e != cudaSuccess) return int(e);
  k_wait_out<<<1, 1, 0, d->stream>>>(d->async_err_dev);
  return int(cudaGetLastError());
}
