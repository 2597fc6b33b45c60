// Operators on caller-owned device buffers: the norm and rotation of query and key heads (qk_norm.cu),
// cross attention to packed states (cross_attn.cu), projections with low-rank adapters (lora.cu).
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/kh_cuda.h"

namespace kh {

void qk_norm_rope(const kh_qk_norm_rope_args* a, cudaStream_t st);
int64_t cross_attention_workspace(const kh_cross_attention_args* a);
void cross_attention(const kh_cross_attention_args* a, cudaStream_t st);
int64_t lora_matmul_workspace(const kh_lora_matmul_args* a);
void lora_matmul(const kh_lora_matmul_args* a, cudaStream_t st);

// Synchronizes `st`; throws all that the operators met on the current device since the last report
// (CudaError where a wait gave up, else ArgError: a position or an adapter id outside its table).
void operator_status(cudaStream_t st);
// Records codes as the operators' kernels would (0: none), in the order of OperatorWord.
void selftest_operator_status(const int (&codes)[4], cudaStream_t st);

// Words in which the operators' kernels leave what they meet, on the current device. A bad index and a wait that
// gave up have a word each, so that neither hides the other.
enum OperatorWord { NORM_INDEX, CROSS_WAIT, LORA_WAIT, LORA_INDEX, OPERATOR_WORDS };
// Bits of an index word (a wait's is the code of the first that gave up).
constexpr int OP_BAD_INDEX = 1;   // a position or an adapter id outside its table
constexpr int OP_BAD_STARTS = 2;  // segment starts that decrease
int* qk_norm_index_word();
int* cross_attention_wait_word();
int* lora_wait_word();
int* lora_index_word();

// Shared argument checks (ArgError with the entry point's name).
void check_that(bool ok, const char* fn, const char* what);
inline bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3) == 0; }
// The stream belongs to the current device.
void check_stream(const char* fn, cudaStream_t st);
// Memory a kernel on the current device can use: device memory of that device, managed or page-locked
// host memory. A pointer of another device or of plain host memory would fault in the kernel.
void check_device_memory(const char* fn, const char* what, const void* p);

}  // namespace kh
