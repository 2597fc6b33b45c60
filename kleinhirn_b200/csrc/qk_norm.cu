// Per-head RMS norm of queries and keys with the position rotation, one pass over the rows.
//
// For a head x of D values with weight w: y = x * rsqrt(mean(x^2) + eps) * w, then for the pairs of
// the first R values (a, b) -> (a c - b s, b c + a s) with the f32 cosine and sine of the row's
// position. Everything between the load and the store is f32; one rounding at the store.
//
// Bound: HBM, each value read and written once (7 operations per value).
// Layout: a head is cut into chunks of VEC values (one load each), and a thread owns two chunks of the
// same head, the pair that the rotation mixes (chunk i and the one R / 2 values on; neighbours when
// the pairs are neighbours or behind R), so the rotation needs no exchange. LANES threads, a power of
// two, hold a head and add their squares by shuffles. A thread takes U heads of the same row, so that
// it loads the angles and weights once, and has 2 U loads in flight.

#include "device_ops.h"

#include <cuda_fp16.h>

#include <algorithm>

#include "runtime.h"
#include "tmap.h"

namespace kh {

namespace {

__device__ int kh_norm_error = 0;

struct NormParams {
  const void* x;
  void* out;
  int64_t rows, x_stride, out_stride, table_rows;
  const float* qw;
  const float* kw;
  const float* cossin;
  const int32_t* positions;
  int q_heads, k_heads, D, R;
  int q_blocks, blocks;  // blocks of U heads of a row: those of q, all
  float eps, inv_d;
  bool interleaved;
};

template <typename T, int VEC>
__device__ __forceinline__ void load_chunk(float (&f)[VEC], const T* p) {
  struct alignas(sizeof(T) * VEC) Raw { T v[VEC]; };
  const Raw r = *reinterpret_cast<const Raw*>(p);
#pragma unroll
  for (int i = 0; i < VEC; ++i) f[i] = float(r.v[i]);
}
template <typename T, int VEC>
__device__ __forceinline__ void store_chunk(T* p, const float (&f)[VEC]) {
  struct alignas(sizeof(T) * VEC) Raw { T v[VEC]; };
  Raw r;
#pragma unroll
  for (int i = 0; i < VEC; ++i) r.v[i] = T(f[i]);
  *reinterpret_cast<Raw*>(p) = r;
}

// PAIRS: chunk pairs of a thread (1, or 4 for the one-value chunks of unaligned heads). LANES * PAIRS
// pairs cover D <= 256.
template <typename T, int VEC, int PAIRS, int U>
__global__ void __launch_bounds__(256) qk_norm_rope_kernel(const NormParams p, int lanes) {
  const int sub = threadIdx.x % lanes;
  const int64_t group = (int64_t(blockIdx.x) * blockDim.x + threadIdx.x) / lanes;
  const int64_t row = group / p.blocks;
  const int block = int(group - row * p.blocks);
  const bool in = row < p.rows;  // (the threads of a head agree; all stay for the shuffles)
  const bool is_k = block >= p.q_blocks;
  const int head0 = (is_k ? block - p.q_blocks : block) * U;
  const int nheads = in ? min(U, (is_k ? p.k_heads : p.q_heads) - head0) : 0;
  const int first = (is_k ? p.q_heads : 0) + head0;  // among all heads of the row

  const int chunks = p.D / VEC;
  const int turned = p.interleaved ? 0 : p.R / 2 / VEC;  // pairs whose chunks lie R / 2 apart
  int c0[PAIRS], c1[PAIRS];
#pragma unroll
  for (int i = 0; i < PAIRS; ++i) {
    const int k = sub + i * lanes;
    c0[i] = k < turned ? k : 2 * k;
    c1[i] = k < turned ? k + turned : 2 * k + 1;
    if (c0[i] >= chunks) c0[i] = -1;
    if (c1[i] >= chunks) c1[i] = -1;
  }

  const T* xr = static_cast<const T*>(p.x) + row * p.x_stride + int64_t(first) * p.D;
  float a[U][PAIRS][VEC], b[U][PAIRS][VEC];
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) a[u][i][e] = b[u][i][e] = 0.f;
      if (u < nheads) {
        if (c0[i] >= 0) load_chunk<T, VEC>(a[u][i], xr + u * p.D + c0[i] * VEC);
        if (c1[i] >= 0) load_chunk<T, VEC>(b[u][i], xr + u * p.D + c1[i] * VEC);
      }
    }

  int64_t pos = 0;
  bool bad = false;
  if (in && p.R) {
    pos = p.positions[row];
    bad = pos < 0 || pos >= p.table_rows;
    if (bad) {
      atomicExch(&kh_norm_error, OP_BAD_INDEX);
      pos = 0;
    }
  }
  const float* cs = p.cossin + pos * 2 * p.R;
  const float* w = is_k ? p.kw : p.qw;

  float scale[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < PAIRS; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) ss += a[u][i][e] * a[u][i][e] + b[u][i][e] * b[u][i][e];
    for (int o = lanes >> 1; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    scale[u] = rsqrtf(ss * p.inv_d + p.eps);
  }

  T* yr = static_cast<T*>(p.out) + row * p.out_stride + int64_t(first) * p.D;
#pragma unroll
  for (int i = 0; i < PAIRS; ++i) {
    if (c0[i] < 0) continue;
    const int d0 = c0[i] * VEC, d1 = c1[i] * VEC;
    float w0[VEC], w1[VEC], c[VEC], s[VEC], ci[VEC], si[VEC];
    // angles: pairs apart use (c, s)[e] for (a[e], b[e]); neighbours inside a chunk use (c, s) for the
    // pairs of a and (ci, si) for those of b
    const bool apart = sub + i * lanes < turned;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      w0[e] = w ? __ldg(w + d0 + e) : 1.f;
      w1[e] = w && c1[i] >= 0 ? __ldg(w + d1 + e) : 1.f;
      c[e] = ci[e] = 1.f;
      s[e] = si[e] = 0.f;
      if (apart) {
        c[e] = __ldg(cs + d0 + e);
        s[e] = __ldg(cs + p.R + d0 + e);
      } else if (p.interleaved) {
        if (d0 + e < p.R) {
          c[e] = __ldg(cs + (d0 + e) / 2);
          s[e] = __ldg(cs + p.R + (d0 + e) / 2);
        }
        if (c1[i] >= 0 && d1 + e < p.R) {
          ci[e] = __ldg(cs + (d1 + e) / 2);
          si[e] = __ldg(cs + p.R + (d1 + e) / 2);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u >= nheads) break;
      float y0[VEC], y1[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        y0[e] = a[u][i][e] * scale[u] * w0[e];
        y1[e] = b[u][i][e] * scale[u] * w1[e];
      }
      if (apart) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float t = y0[e] * c[e] - y1[e] * s[e];
          y1[e] = y1[e] * c[e] + y0[e] * s[e];
          y0[e] = t;
        }
      } else if (p.interleaved) {
        if constexpr (VEC == 1) {  // the pair is the two one-value chunks
          const float t = y0[0] * c[0] - y1[0] * s[0];
          y1[0] = y1[0] * c[0] + y0[0] * s[0];
          y0[0] = t;
        } else {
#pragma unroll
          for (int e = 0; e < VEC; e += 2) {
            const float t = y0[e] * c[e] - y0[e + 1] * s[e];
            y0[e + 1] = y0[e + 1] * c[e] + y0[e] * s[e];
            y0[e] = t;
            const float r = y1[e] * ci[e] - y1[e + 1] * si[e];
            y1[e + 1] = y1[e + 1] * ci[e] + y1[e] * si[e];
            y1[e] = r;
          }
        }
      }
      if (bad) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) y0[e] = y1[e] = 0.f;
      }
      store_chunk<T, VEC>(yr + u * p.D + d0, y0);
      if (c1[i] >= 0) store_chunk<T, VEC>(yr + u * p.D + d1, y1);
    }
  }
}

template <typename T, int VEC, int PAIRS, int U>
void launch(NormParams p, cudaStream_t st) {
  const int pairs = (p.D / VEC + 1) / 2;
  int lanes = 1;
  while (lanes * PAIRS < pairs) lanes *= 2;
  p.q_blocks = (p.q_heads + U - 1) / U;
  p.blocks = p.q_blocks + (p.k_heads + U - 1) / U;
  const int64_t threads = p.rows * p.blocks * lanes;
  const int64_t grid = (threads + 255) / 256;
  check_that(grid < (int64_t(1) << 31), "kh_qk_norm_rope", "rows * heads too large");
  qk_norm_rope_kernel<T, VEC, PAIRS, U><<<unsigned(grid), 256, 0, st>>>(p, lanes);
  KH_CUDA(cudaGetLastError());
}

// Whether chunks of `vec` values fit the head, its rotation and every row's alignment.
bool fits(const kh_qk_norm_rope_args& a, int size, int vec) {
  const uintptr_t bytes = uintptr_t(vec) * size;
  return a.head_dim % vec == 0 && (a.interleaved || (a.rotary_dim / 2) % vec == 0) &&
         reinterpret_cast<uintptr_t>(a.x) % bytes == 0 && reinterpret_cast<uintptr_t>(a.out) % bytes == 0 &&
         a.x_stride % vec == 0 && a.out_stride % vec == 0;
}

}  // namespace

void qk_norm_rope(const kh_qk_norm_rope_args* args, cudaStream_t st) {
  const char* fn = "kh_qk_norm_rope";
  check_that(args != nullptr, fn, "null arguments");
  const kh_qk_norm_rope_args& a = *args;
  check_that(a.dtype == KH_F32 || a.dtype == KH_F16, fn, "dtype must be KH_F32 or KH_F16");
  check_that(a.head_dim >= 2 && a.head_dim <= 256 && a.head_dim % 2 == 0, fn, "head_dim must be even, in [2, 256]");
  check_that(a.rotary_dim >= 0 && a.rotary_dim <= a.head_dim && a.rotary_dim % 2 == 0, fn,
             "rotary_dim must be even, in [0, head_dim]");
  check_that(a.q_heads >= 0 && a.k_heads >= 0 && a.q_heads <= 4096 && a.k_heads <= 4096 &&
                 a.q_heads + a.k_heads >= 1 && a.q_heads + a.k_heads <= 4096,
             fn, "q_heads + k_heads must be in [1, 4096]");
  check_that(a.interleaved == 0 || a.interleaved == 1, fn, "interleaved must be 0 or 1");
  check_that(a.eps > 0.f, fn, "eps must be above 0");
  check_that(a.rows >= 0 && a.rows < (int64_t(1) << 40), fn, "rows must be in [0, 2^40)");
  const int64_t width = int64_t(a.q_heads + a.k_heads) * a.head_dim;
  check_that(a.x_stride >= width && a.out_stride >= width && a.x_stride < (int64_t(1) << 31) &&
                 a.out_stride < (int64_t(1) << 31),
             fn, "strides must be at least (q_heads + k_heads) * head_dim and below 2^31");
  if (a.rows == 0) return;
  const int size = a.dtype == KH_F16 ? 2 : 4;
  check_that(a.x && a.out, fn, "null x or out");
  check_that(reinterpret_cast<uintptr_t>(a.x) % size == 0 && reinterpret_cast<uintptr_t>(a.out) % size == 0, fn,
             "x and out must be aligned to their values");
  // rows of an in-place call are read and written by the same threads; any other overlap is a race
  const char *xb = static_cast<const char*>(a.x), *ob = static_cast<const char*>(a.out);
  const int64_t x_end = ((a.rows - 1) * a.x_stride + width) * size, o_end = ((a.rows - 1) * a.out_stride + width) * size;
  check_that((xb == ob && a.x_stride == a.out_stride) || xb + x_end <= ob || ob + o_end <= xb ||
                 // two column blocks of the same rows
                 (a.x_stride == a.out_stride && (ob > xb ? ob - xb : xb - ob) % (a.x_stride * size) >= width * size &&
                  (ob > xb ? ob - xb : xb - ob) % (a.x_stride * size) <= (a.x_stride - width) * size),
             fn, "out overlaps x (it may be x itself, with the same stride)");
  if (a.rotary_dim) {
    check_that(a.cossin && a.positions, fn, "null cossin or positions");
    check_that(a.table_rows >= 1, fn, "table_rows must be at least 1");
    check_that(reinterpret_cast<uintptr_t>(a.cossin) % 4 == 0 && reinterpret_cast<uintptr_t>(a.positions) % 4 == 0,
               fn, "cossin and positions must be 4-byte aligned");
  }
  check_that(reinterpret_cast<uintptr_t>(a.q_weight) % 4 == 0 && reinterpret_cast<uintptr_t>(a.k_weight) % 4 == 0, fn,
             "weights must be 4-byte aligned");
  check_stream(fn, st);
  check_device_memory(fn, "x", a.x);
  check_device_memory(fn, "out", a.out);
  if (a.q_weight) check_device_memory(fn, "q_weight", a.q_weight);
  if (a.k_weight) check_device_memory(fn, "k_weight", a.k_weight);
  if (a.rotary_dim) {
    check_device_memory(fn, "cossin", a.cossin);
    check_device_memory(fn, "positions", a.positions);
  }
  NormParams p{};
  p.x = a.x;
  p.out = a.out;
  p.rows = a.rows;
  p.x_stride = a.x_stride;
  p.out_stride = a.out_stride;
  p.table_rows = a.table_rows;
  p.qw = a.q_weight;
  p.kw = a.k_weight;
  p.cossin = a.cossin;
  p.positions = a.positions;
  p.q_heads = a.q_heads;
  p.k_heads = a.k_heads;
  p.D = a.head_dim;
  p.R = a.rotary_dim;
  p.eps = a.eps;
  p.inv_d = 1.f / float(a.head_dim);
  p.interleaved = a.interleaved != 0;
  if (a.dtype == KH_F16) {
    if (fits(a, 2, 8)) launch<__half, 8, 1, 2>(p, st);
    else if (fits(a, 2, 4)) launch<__half, 4, 1, 2>(p, st);
    else launch<__half, 1, 4, 1>(p, st);
  } else {
    if (fits(a, 4, 4)) launch<float, 4, 1, 2>(p, st);
    else launch<float, 1, 4, 1>(p, st);
  }
}

int qk_norm_error_code() {
  int v = 0;
  KH_CUDA(cudaMemcpyFromSymbol(&v, kh_norm_error, sizeof(int)));
  if (v) {
    const int zero = 0;
    KH_CUDA(cudaMemcpyToSymbol(kh_norm_error, &zero, sizeof(int)));
  }
  return v;
}

}  // namespace kh
