// What the operators on caller-owned device buffers share: argument checks and the status report.

#include "device_ops.h"

#include <string>

#include "runtime.h"
#include "tmap.h"

namespace kh {

void check_that(bool ok, const char* fn, const char* what) {
  if (!ok) throw ArgError(std::string(fn) + ": " + what);
}

void check_stream(const char* fn, cudaStream_t st) {
  if (!st) return;
  // a capturing stream may not be asked (a launch on another device's stream fails with a status)
  cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
  KH_CUDA(cudaStreamIsCapturing(st, &cap));
  if (cap != cudaStreamCaptureStatusNone) return;
  int dev = -1;
  KH_CUDA(cudaStreamGetDevice(st, &dev));
  if (dev != current_device())
    throw ArgError(std::string(fn) + ": the stream belongs to device " + std::to_string(dev) +
                   ", the current device is " + std::to_string(current_device()));
}

void check_device_memory(const char* fn, const char* what, const void* p) {
  cudaPointerAttributes at{};
  KH_CUDA(cudaPointerGetAttributes(&at, p));
  if (at.type == cudaMemoryTypeUnregistered)
    throw ArgError(std::string(fn) + ": " + what + " is not device memory");
  if (at.type == cudaMemoryTypeDevice && at.device != current_device())
    throw ArgError(std::string(fn) + ": " + what + " is memory of device " + std::to_string(at.device) +
                   ", the current device is " + std::to_string(current_device()));
}

void operator_status(cudaStream_t st) {
  check_stream("kh_operator_status", st);
  KH_CUDA(cudaStreamSynchronize(st));
  const int norm = qk_norm_error_code(), cross = cross_attention_error_code(), lora = lora_error_code();
  if (cross) throw CudaError("kh_cross_attention_f16: pipeline wait timed out (code " + std::to_string(cross) + ")");
  if (lora && lora != OP_BAD_INDEX)
    throw CudaError("kh_lora_matmul_f16: pipeline wait timed out (code " + std::to_string(lora) + ")");
  if (norm) throw ArgError("kh_qk_norm_rope: a position outside [0, table_rows)");
  if (lora) throw ArgError("kh_lora_matmul_f16: an adapter id of n_adapters or more");
}

}  // namespace kh
