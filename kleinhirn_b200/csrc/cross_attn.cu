// Cross attention of packed query rows over an encoder's packed states of another length.
//
// For query row i of sequence s and query head h, with g = q_heads / kv_heads and the kept states K of
// s: out = sum_j p_j v_j, p = softmax over j in K of scale q_i,h . k_j,h/g; zero where K is empty.
//
// One warp per (query row, head): the warp walks the states with the running maximum m and sum l of
// the exponentials, its lanes hold D / 32 values of the row each.

#include "device_ops.h"

#include <cuda_fp16.h>

#include <algorithm>

#include "runtime.h"
#include "sm100.cuh"
#include "tmap.h"

namespace kh {

namespace {

using namespace sm100;

struct CrossParams {
  const __half* q;
  const __half* k;
  const __half* v;
  __half* out;
  const float* mask;
  const int32_t* q_starts;
  const int32_t* k_starts;
  int64_t q_rows, kv_rows, q_stride, k_stride, v_stride, out_stride;
  int n_seqs, q_heads, kv_heads, max_q, max_k;
  float scale;
};

// Rows of sequence s in a buffer of `rows`: starts outside it are cut, a longer sequence ends at `most`.
__device__ __forceinline__ void seq_range(const int32_t* starts, int s, int64_t rows, int most, int64_t& r0, int& n) {
  r0 = min(max(int64_t(starts[s]), int64_t(0)), rows);
  const int64_t r1 = min(max(int64_t(starts[s + 1]), r0), rows);
  n = int(min(r1 - r0, int64_t(most)));
}

template <int D>
__global__ void __launch_bounds__(128) cross_simple_kernel(const CrossParams p) {
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31;
  const int s = blockIdx.z, h = blockIdx.y;
  const int i = blockIdx.x * 4 + (threadIdx.x >> 5);
  int64_t q0, k0;
  int nq, nk;
  seq_range(p.q_starts, s, p.q_rows, p.max_q, q0, nq);
  seq_range(p.k_starts, s, p.kv_rows, p.max_k, k0, nk);
  if (i >= nq) return;
  const int hk = h / (p.q_heads / p.kv_heads);
  float q[E], o[E], m = -INFINITY, l = 0.f;
  for (int e = 0; e < E; ++e) {
    q[e] = __half2float(p.q[(q0 + i) * p.q_stride + h * D + e * 32 + lane]) * p.scale;
    o[e] = 0.f;
  }
  for (int j = 0; j < nk; ++j) {
    if (p.mask && !(p.mask[k0 + j] > 0.5f)) continue;
    float d = 0.f;
    for (int e = 0; e < E; ++e) d += q[e] * __half2float(p.k[(k0 + j) * p.k_stride + hk * D + e * 32 + lane]);
    for (int w = 16; w; w >>= 1) d += __shfl_xor_sync(0xffffffffu, d, w);
    const float mn = fmaxf(m, d);
    const float c = mn == -INFINITY ? 1.f : expf(m - mn), x = mn == -INFINITY ? 0.f : expf(d - mn);
    m = mn;
    l = l * c + x;
    for (int e = 0; e < E; ++e)
      o[e] = o[e] * c + x * __half2float(p.v[(k0 + j) * p.v_stride + hk * D + e * 32 + lane]);
  }
  for (int e = 0; e < E; ++e)
    p.out[(q0 + i) * p.out_stride + h * D + e * 32 + lane] = __float2half_rn(l > 0.f ? o[e] / l : l);
}

void check_sizes(const char* fn, const kh_cross_attention_args* args) {
  check_that(args != nullptr, fn, "null arguments");
  const kh_cross_attention_args& a = *args;
  check_that(a.n_seqs >= 0 && a.n_seqs <= 65535, fn, "n_seqs must be in [0, 65535]");
  check_that(a.head_dim == 32 || a.head_dim == 64 || a.head_dim == 128, fn, "head_dim must be 32, 64 or 128");
  check_that(a.q_heads >= 1 && a.q_heads <= 1024 && a.kv_heads >= 1 && a.q_heads % a.kv_heads == 0 &&
                 a.q_heads / a.kv_heads <= 64,
             fn, "q_heads must be in [1, 1024], a multiple of kv_heads, at most 64 to one");
  check_that(a.max_q >= 0 && a.max_k >= 0 && a.max_q <= (1 << 24) && a.max_k <= (1 << 24), fn,
             "max_q and max_k must be in [0, 2^24]");
  check_that(a.q_rows >= 0 && a.q_rows < (int64_t(1) << 31) && a.kv_rows >= 0 && a.kv_rows < (int64_t(1) << 31), fn,
             "q_rows and kv_rows must be in [0, 2^31)");
}

}  // namespace

int64_t cross_attention_workspace(const kh_cross_attention_args* args) {
  check_sizes("kh_cross_attention_f16_workspace", args);
  return 0;
}

void cross_attention(const kh_cross_attention_args* args, cudaStream_t st) {
  const char* fn = "kh_cross_attention_f16";
  check_sizes(fn, args);
  const kh_cross_attention_args& a = *args;
  if (a.n_seqs == 0 || a.max_q == 0 || a.q_rows == 0) return;
  const bool states = a.kv_rows > 0 && a.max_k > 0;
  auto aligned = [](const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15) == 0; };
  check_that(a.q && a.out && a.q_starts && a.k_starts && (!states || (a.k && a.v)), fn, "null pointer argument");
  check_that(aligned(a.q) && aligned(a.out) && aligned(a.k) && aligned(a.v), fn,
             "q, k, v and out must be 16-byte aligned");
  const int64_t qw = int64_t(a.q_heads) * a.head_dim, kw = int64_t(a.kv_heads) * a.head_dim;
  const int64_t lim = int64_t(1) << 31;
  check_that(a.q_stride >= qw && a.out_stride >= qw && a.q_stride < lim && a.out_stride < lim &&
                 (!states || (a.k_stride >= kw && a.v_stride >= kw && a.k_stride < lim && a.v_stride < lim)),
             fn, "a stride is shorter than its rows (or 2^31 and more)");
  check_that(a.q_stride % 8 == 0 && a.out_stride % 8 == 0 && a.k_stride % 8 == 0 && a.v_stride % 8 == 0, fn,
             "strides must be multiples of 8");
  const int64_t need = cross_attention_workspace(args);
  check_that(need == 0 || (a.workspace && int64_t(a.workspace_bytes) >= need), fn, "workspace too small");
  check_that((reinterpret_cast<uintptr_t>(a.workspace) & 255) == 0, fn, "workspace must be 256-byte aligned");
  check_stream(fn, st);
  check_device_memory(fn, "q", a.q);
  check_device_memory(fn, "out", a.out);
  check_device_memory(fn, "q_starts", a.q_starts);
  check_device_memory(fn, "k_starts", a.k_starts);
  if (states) {
    check_device_memory(fn, "k", a.k);
    check_device_memory(fn, "v", a.v);
    if (a.key_mask) check_device_memory(fn, "key_mask", a.key_mask);
  }
  if (need) check_device_memory(fn, "workspace", a.workspace);
  CrossParams p{};
  p.q = static_cast<const __half*>(a.q);
  p.k = static_cast<const __half*>(a.k);
  p.v = static_cast<const __half*>(a.v);
  p.out = static_cast<__half*>(a.out);
  p.mask = a.key_mask;
  p.q_starts = a.q_starts;
  p.k_starts = a.k_starts;
  p.q_rows = a.q_rows;
  p.kv_rows = states ? a.kv_rows : 0;
  p.q_stride = a.q_stride;
  p.k_stride = a.k_stride;
  p.v_stride = a.v_stride;
  p.out_stride = a.out_stride;
  p.n_seqs = a.n_seqs;
  p.q_heads = a.q_heads;
  p.kv_heads = a.kv_heads;
  p.max_q = a.max_q;
  p.max_k = a.max_k;
  p.scale = a.scale;
  const dim3 grid((a.max_q + 3) / 4, a.q_heads, a.n_seqs);
  if (a.head_dim == 32) cross_simple_kernel<32><<<grid, 128, 0, st>>>(p);
  else if (a.head_dim == 64) cross_simple_kernel<64><<<grid, 128, 0, st>>>(p);
  else cross_simple_kernel<128><<<grid, 128, 0, st>>>(p);
  KH_CUDA(cudaGetLastError());
}

int cross_attention_error_code() {
  int v = 0;
  KH_CUDA(cudaMemcpyFromSymbol(&v, sm100::kh_tc_error, sizeof(int)));
  if (v) {
    const int zero = 0;
    KH_CUDA(cudaMemcpyToSymbol(sm100::kh_tc_error, &zero, sizeof(int)));
  }
  return v;
}

}  // namespace kh
