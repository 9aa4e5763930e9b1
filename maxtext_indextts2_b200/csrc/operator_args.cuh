// Checks of the arguments of the operators that stand alone (fp8_linear.cu, logit_controls.cu).
#pragma once

#include <initializer_list>

#include "host_util.cuh"

namespace {

// Kernels run on the current device: memory of another one, or of the host alone, would fault in them.  (0.1 us per pointer; legal while a stream is captured)
int on_this_device(std::initializer_list<const void*> pointers) {
  int device;
  MTX_CUDA(cudaGetDevice(&device));
  for (const void* p : pointers) {
    if (p == nullptr) continue;  // (a part that is left out)
    cudaPointerAttributes a;
    MTX_CUDA(cudaPointerGetAttributes(&a, p));
    if (a.type == cudaMemoryTypeUnregistered) return fail(MTX_ERR_ARG, "%p is not device memory", p);
    if (a.type == cudaMemoryTypeDevice && a.device != device) return fail(MTX_ERR_ARG, "%p is memory of device %d; the current device is %d", p, a.device, device);
  }
  return MTX_OK;
}

}  // namespace
