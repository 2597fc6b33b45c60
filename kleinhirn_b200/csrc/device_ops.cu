// What the operators on caller-owned device buffers share: argument checks and the status report.

#include "device_ops.h"

#include <algorithm>
#include <mutex>
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

namespace {

struct Words {
  int* at[OPERATOR_WORDS];
};
Words operator_words() {
  Words w{};
  w.at[NORM_INDEX] = qk_norm_index_word();
  w.at[CROSS_WAIT] = cross_attention_wait_word();
  w.at[LORA_WAIT] = lora_wait_word();
  w.at[LORA_INDEX] = lora_index_word();
  return w;
}

struct Codes {
  int v[OPERATOR_WORDS];
};
__device__ Codes kh_taken;

// Reads and clears each word at once: what a kernel on another stream adds meanwhile stays for the next report.
__global__ void take_words_kernel(Words w) { kh_taken.v[threadIdx.x] = atomicExch(w.at[threadIdx.x], 0); }
__global__ void add_codes_kernel(Words w, Codes c) { atomicCAS(w.at[threadIdx.x], 0, c.v[threadIdx.x]); }

}  // namespace

void operator_status(cudaStream_t st) {
  const char* fn = "kh_operator_status";
  cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
  const cudaError_t asked = cudaStreamIsCapturing(st, &cap);
  if (asked == cudaErrorStreamCaptureImplicit) (void)cudaGetLastError();  // the legacy stream beside a capture
  else KH_CUDA(asked);
  check_that(asked == cudaSuccess && cap == cudaStreamCaptureStatusNone, fn, "not while a capture is under way");
  check_stream(fn, st);
  KH_CUDA(cudaStreamSynchronize(st));
  Codes c{};
  {
    static std::mutex one;  // kh_taken serves one report at a time
    std::lock_guard<std::mutex> lock(one);
    void* taken = nullptr;
    KH_CUDA(cudaGetSymbolAddress(&taken, kh_taken));
    take_words_kernel<<<1, OPERATOR_WORDS, 0, st>>>(operator_words());
    KH_CUDA(cudaGetLastError());
    KH_CUDA(cudaMemcpyAsync(&c, taken, sizeof c, cudaMemcpyDeviceToHost, st));
    KH_CUDA(cudaStreamSynchronize(st));
  }
  std::string met;
  auto add = [&](const std::string& what) { met += (met.empty() ? "" : "; ") + what; };
  auto wait = [&](const char* op, int code) {
    if (code) add(std::string(op) + ": pipeline wait timed out (code " + std::to_string(code) + ")");
  };
  wait("kh_cross_attention_f16", c.v[CROSS_WAIT]);
  wait("kh_lora_matmul_f16", c.v[LORA_WAIT]);
  if (c.v[NORM_INDEX]) add("kh_qk_norm_rope: a position outside [0, table_rows)");
  if (c.v[LORA_INDEX] & OP_BAD_INDEX) add("kh_lora_matmul_f16: an adapter id of n_adapters or more");
  if (c.v[LORA_INDEX] & OP_BAD_STARTS) add("kh_lora_matmul_f16: segment starts that decrease (some rows are without their adapter)");
  if (c.v[CROSS_WAIT] || c.v[LORA_WAIT]) throw CudaError(met);
  if (!met.empty()) throw ArgError(met);
}

void selftest_operator_status(const int (&codes)[4], cudaStream_t st) {
  static_assert(OPERATOR_WORDS == 4, "one code a word");
  check_stream("kh_selftest_operator_status", st);
  Codes c{};
  std::copy(codes, codes + 4, c.v);
  add_codes_kernel<<<1, OPERATOR_WORDS, 0, st>>>(operator_words(), c);
  KH_CUDA(cudaGetLastError());
}

}  // namespace kh
