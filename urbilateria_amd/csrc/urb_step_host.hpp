// urb_step_host.hpp -- what the C ABIs of the decoder steps and of the paged cache share: checks and the
// status word of a context.
#pragma once

#include "../../include/urb_moe.h"

#include <hip/hip_runtime.h>

#include <utility>

#include "urb_kernels.hpp"

#define URB_HIP(call)                            \
  do {                                           \
    hipError_t e_ = (call);                      \
    if (e_ == hipErrorOutOfMemory) return URB_ERR_OUT_OF_MEMORY; \
    if (e_ != hipSuccess) return URB_ERR_DEVICE; \
  } while (0)

namespace {

constexpr size_t kAlign = 256;
size_t align_up(size_t v) { return (v + kAlign - 1) / kAlign * kAlign; }

bool row_type(urb_dtype t) { return t == URB_DTYPE_BF16 || t == URB_DTYPE_F32; }
size_t value_bytes(urb_dtype t) { return t == URB_DTYPE_BF16 ? 2 : 4; }
bool finite_host(float v) { return v == v && v <= 3.4028235e38f && v >= -3.4028235e38f; }

bool on_device(int device) {
  int now = -1;
  return hipGetDevice(&now) == hipSuccess && now == device;
}

// Whether the heads of an output lie apart: [tokens][heads] rows of dim values, either stride the larger.
bool heads_apart(uint64_t tokens, uint64_t token_stride, uint64_t heads, uint64_t head_stride, uint64_t dim) {
  if (token_stride < head_stride) {
    std::swap(tokens, heads);
    std::swap(token_stride, head_stride);
  }
  if (heads > 1 && head_stride < dim) return false;
  if (tokens == 1) return true;
  // (the larger stride against what the others span, without the product)
  return token_stride >= dim && (heads == 1 || (token_stride - dim) / (heads - 1) >= head_stride);
}

// Waits for the stream, then reads and clears a status word (written by kernels of that stream).
urb_status take_status(int* word, hipStream_t s, int* bits) {
  *bits = 0;
  URB_HIP(hipStreamSynchronize(s));
  URB_HIP(hipMemcpy(bits, word, sizeof(int), hipMemcpyDeviceToHost));
  urb::launch_fill_i32(word, 0, 1, s);
  URB_HIP(hipGetLastError());
  URB_HIP(hipStreamSynchronize(s));
  return URB_OK;
}

}  // namespace
