// Checks of the arguments, and launches, of the operators that stand alone (fp8_linear.cu, logit_controls.cu, row_operators.cu, prefix_attention.cu, verify_drafts.cu).
#pragma once

#include <initializer_list>

#include "host_util.cuh"

namespace {

// Whether what is there lies on multiples of `bytes`: a load of its type would fault otherwise.
bool lie_on(size_t bytes, std::initializer_list<const void*> pointers) {
  for (const void* p : pointers)
    if (reinterpret_cast<uintptr_t>(p) % bytes != 0) return false;
  return true;
}

// Kernels run on the current device: memory of another one, or of the host alone, would fault in them.  pinned: host memory that the device can read is one of
// the arguments' places.  (0.07 us per pointer; legal while a stream is captured)
int on_this_device(std::initializer_list<const void*> pointers, bool pinned = false) {
  int device;
  MTX_CUDA(cudaGetDevice(&device));
  for (const void* p : pointers) {
    if (p == nullptr) continue;  // (a part that is left out)
    cudaPointerAttributes a;
    MTX_CUDA(cudaPointerGetAttributes(&a, p));
    if (a.type == cudaMemoryTypeUnregistered || (a.type == cudaMemoryTypeHost && !pinned)) return fail(MTX_ERR_ARG, "%p is not device memory", p);
    if (a.type == cudaMemoryTypeDevice && a.device != device) return fail(MTX_ERR_ARG, "%p is memory of device %d; the current device is %d", p, a.device, device);
  }
  return MTX_OK;
}

// a kernel's opt-in to more shared memory, once per device
template <class Kernel>
int allow_smem(Kernel kernel, size_t bytes, std::atomic<uint64_t>& done) {
  int device;
  MTX_CUDA(cudaGetDevice(&device));
  const uint64_t bit = 1ull << (device & 63);
  if ((done.load(std::memory_order_relaxed) & bit) == 0) {
    MTX_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes)));
    done.fetch_or(bit, std::memory_order_relaxed);
  }
  return MTX_OK;
}

}  // namespace
