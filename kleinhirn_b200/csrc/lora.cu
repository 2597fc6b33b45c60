// A projection with the low-rank adapters of many requests.
//
// out[t] = x[t] W^T + bias + s_a (x[t] A_a^T) B_a^T, a the adapter of the segment of rows that t lies
// in. Two steps: h[t] = s_a x[t] A_a^T (rank values a row, rounded to f16: its rounding is 2^-11 of the
// adapter's own part, as far below the output's as that part is below the projection), then the
// projection and h B_a^T into the same f32 sum, rounded once.

#include "device_ops.h"

#include <cuda_fp16.h>

#include <algorithm>

#include "runtime.h"
#include "sm100.cuh"
#include "tmap.h"

namespace kh {

namespace {

using namespace sm100;

struct LoraParams {
  const __half* x;
  const __half* w;
  const __half* bias;
  const __half* a;
  const __half* b;
  const float* scales;
  const int32_t* starts;
  const int32_t* ids;
  __half* out;
  __half* h;
  int64_t rows, x_stride, out_stride;
  int k, n, rank, n_adapters, n_segs;
};

// Start of segment i, cut to the buffer.
__device__ __forceinline__ int64_t seg_start(const LoraParams& p, int i) {
  return min(max(int64_t(p.starts[i]), int64_t(0)), p.rows);
}
// Segment of row t (the last one that starts at or before it), or -1 before the first and behind the last.
__device__ __forceinline__ int seg_of(const LoraParams& p, int64_t t) {
  if (t < seg_start(p, 0) || t >= seg_start(p, p.n_segs)) return -1;
  int lo = 0, hi = p.n_segs - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (seg_start(p, mid) <= t) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}
// Adapter of a segment, -1 for none; an id that does not exist counts as none and is reported.
__device__ __forceinline__ int adapter_of(const LoraParams& p, int seg) {
  const int a = p.ids[seg];
  if (a < p.n_adapters) return a < 0 ? -1 : a;
  atomicCAS(&kh_tc_error, 0, OP_BAD_INDEX);
  return -1;
}

// One warp per (row, rank index).
__global__ void __launch_bounds__(256) lora_shrink_simple_kernel(const LoraParams p) {
  const int64_t t = blockIdx.x;
  const int lane = threadIdx.x & 31;
  const int seg = seg_of(p, t);
  if (seg < 0) return;
  const int a = adapter_of(p, seg);
  if (a < 0) return;
  for (int r = threadIdx.x >> 5; r < p.rank; r += 8) {
    float d = 0.f;
    for (int i = lane; i < p.k; i += 32)
      d += __half2float(p.x[t * p.x_stride + i]) * __half2float(p.a[(int64_t(a) * p.rank + r) * p.k + i]);
    for (int o = 16; o; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
    if (lane == 0) p.h[t * p.rank + r] = __float2half_rn(d * (p.scales ? p.scales[a] : 1.f));
  }
}

// 64 x 64 outputs of a CTA, 4 x 4 of a thread.
__global__ void __launch_bounds__(256) lora_simple_kernel(const LoraParams p) {
  __shared__ float xs[64][17], ws[64][17];
  const int64_t t0 = int64_t(blockIdx.x) * 64;
  const int n0 = blockIdx.y * 64, ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  float acc[4][4] = {};
  for (int k0 = 0; k0 < p.k; k0 += 16) {
    for (int i = threadIdx.x; i < 1024; i += 256) {
      const int r = i / 16, c = i % 16;
      xs[r][c] = t0 + r < p.rows && k0 + c < p.k ? __half2float(p.x[(t0 + r) * p.x_stride + k0 + c]) : 0.f;
      ws[r][c] = n0 + r < p.n && k0 + c < p.k ? __half2float(p.w[int64_t(n0 + r) * p.k + k0 + c]) : 0.f;
    }
    __syncthreads();
    for (int c = 0; c < 16; ++c)
      for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) acc[i][j] += xs[ty + 16 * i][c] * ws[tx + 16 * j][c];
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i) {
    const int64_t t = t0 + ty + 16 * i;
    const int seg = t < p.rows ? seg_of(p, t) : -1;
    if (seg < 0) continue;
    const int a = adapter_of(p, seg);
    for (int j = 0; j < 4; ++j) {
      const int n = n0 + tx + 16 * j;
      if (n >= p.n) continue;
      float v = acc[i][j];
      if (a >= 0)
        for (int r = 0; r < p.rank; ++r)
          v += __half2float(p.h[t * p.rank + r]) * __half2float(p.b[(int64_t(a) * p.n + n) * p.rank + r]);
      if (p.bias) v += __half2float(p.bias[n]);
      p.out[t * p.out_stride + n] = __float2half_rn(v);
    }
  }
}

void check_sizes(const char* fn, const kh_lora_matmul_args* args) {
  check_that(args != nullptr, fn, "null arguments");
  const kh_lora_matmul_args& a = *args;
  check_that(a.k >= 8 && a.k <= 65536 && a.k % 8 == 0 && a.n >= 8 && a.n <= 65536 && a.n % 8 == 0, fn,
             "k and n must be multiples of 8, in [8, 65536]");
  check_that(a.rank >= 8 && a.rank <= 128 && a.rank % 8 == 0, fn, "rank must be a multiple of 8, in [8, 128]");
  check_that(a.n_adapters >= 0 && a.n_adapters <= 65535, fn, "n_adapters must be in [0, 65535]");
  check_that(a.n_segs >= 0 && a.n_segs <= 65535, fn, "n_segs must be in [0, 65535]");
  check_that(a.rows >= 0 && a.rows < (int64_t(1) << 31) - 256, fn, "rows must be in [0, 2^31 - 256)");
}

}  // namespace

int64_t lora_matmul_workspace(const kh_lora_matmul_args* args) {
  check_sizes("kh_lora_matmul_f16_workspace", args);
  return args->rows * args->rank * 2;
}

void lora_matmul(const kh_lora_matmul_args* args, cudaStream_t st) {
  const char* fn = "kh_lora_matmul_f16";
  check_sizes(fn, args);
  const kh_lora_matmul_args& a = *args;
  if (a.n_segs == 0 || a.rows == 0) return;
  auto aligned = [](const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15) == 0; };
  check_that(a.x && a.w && a.out && a.seg_starts && a.seg_adapters && (a.n_adapters == 0 || (a.lora_a && a.lora_b)), fn,
             "null pointer argument");
  check_that(aligned(a.x) && aligned(a.w) && aligned(a.bias) && aligned(a.lora_a) && aligned(a.lora_b) &&
                 aligned(a.out),
             fn, "x, w, bias, lora_a, lora_b and out must be 16-byte aligned");
  const int64_t lim = int64_t(1) << 31;
  check_that(a.x_stride >= a.k && a.out_stride >= a.n && a.x_stride < lim && a.out_stride < lim &&
                 a.x_stride % 8 == 0 && a.out_stride % 8 == 0,
             fn, "strides must be multiples of 8, at least k and n, below 2^31");
  const int64_t need = lora_matmul_workspace(args);
  check_that(need == 0 || (a.workspace && int64_t(a.workspace_bytes) >= need), fn, "workspace too small");
  check_that((reinterpret_cast<uintptr_t>(a.workspace) & 255) == 0, fn, "workspace must be 256-byte aligned");
  check_stream(fn, st);
  check_device_memory(fn, "x", a.x);
  check_device_memory(fn, "w", a.w);
  check_device_memory(fn, "out", a.out);
  check_device_memory(fn, "seg_starts", a.seg_starts);
  check_device_memory(fn, "seg_adapters", a.seg_adapters);
  if (a.bias) check_device_memory(fn, "bias", a.bias);
  if (a.n_adapters) {
    check_device_memory(fn, "lora_a", a.lora_a);
    check_device_memory(fn, "lora_b", a.lora_b);
    if (a.scales) check_device_memory(fn, "scales", a.scales);
  }
  if (need) check_device_memory(fn, "workspace", a.workspace);
  LoraParams p{};
  p.x = static_cast<const __half*>(a.x);
  p.w = static_cast<const __half*>(a.w);
  p.bias = static_cast<const __half*>(a.bias);
  p.a = static_cast<const __half*>(a.lora_a);
  p.b = static_cast<const __half*>(a.lora_b);
  p.scales = a.scales;
  p.starts = a.seg_starts;
  p.ids = a.seg_adapters;
  p.out = static_cast<__half*>(a.out);
  p.h = static_cast<__half*>(a.workspace);
  p.rows = a.rows;
  p.x_stride = a.x_stride;
  p.out_stride = a.out_stride;
  p.k = a.k;
  p.n = a.n;
  p.rank = a.rank;
  p.n_adapters = a.n_adapters;
  p.n_segs = a.n_segs;
  lora_shrink_simple_kernel<<<unsigned(a.rows), 256, 0, st>>>(p);
  const dim3 grid(unsigned((a.rows + 63) / 64), unsigned((a.n + 63) / 64));
  lora_simple_kernel<<<grid, 256, 0, st>>>(p);
  KH_CUDA(cudaGetLastError());
}

int lora_error_code() {
  int v = 0;
  KH_CUDA(cudaMemcpyFromSymbol(&v, sm100::kh_tc_error, sizeof(int)));
  if (v) {
    const int zero = 0;
    KH_CUDA(cudaMemcpyToSymbol(sm100::kh_tc_error, &zero, sizeof(int)));
  }
  return v;
}

}  // namespace kh
