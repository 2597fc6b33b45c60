// Per-head RMS norm of queries and keys with the position rotation, one pass over the rows.
//
// For a head x of D values with weight w: y = x * rsqrt(mean(x^2) + eps) * w, then for the pairs of
// the first R values (a, b) -> (a c - b s, b c + a s) with the f32 cosine and sine of the row's
// position. Everything between the load and the store is f32; one rounding at the store.
//
// Bound: HBM, each value read and written once (7 operations per value).
// Layout: a head is cut into chunks of VEC values (one load each). In the usual kernel a thread owns one chunk and
// takes the chunk that the rotation mixes with it from that chunk's lane; in the one for other heads it owns both,
// and the rotation needs no exchange. The threads of a head add their squares by shuffles. A thread takes U heads
// of the same row: it loads the angles and weights once, folds them into coefficients w cos and w sin (the scale
// of a head comes last), and has the loads of all its heads in flight.

#include "device_ops.h"

#include <cuda_fp16.h>

#include <algorithm>

#include "runtime.h"
#include "sm100.cuh"
#include "tmap.h"

namespace kh {

namespace {

__device__ int kh_norm_error = 0;

struct NormParams {
  const void* x;
  void* out;
  int64_t x_stride, out_stride, table_rows;
  const float* qw;
  const float* kw;
  const float* cossin;
  const int32_t* positions;
  uint32_t groups;  // rows * blocks of this launch
  int q_heads, k_heads, D, R;
  uint32_t q_blocks, blocks;  // blocks of U heads of a row: those of q, all
  uint32_t lane_inv;          // 1024 / chunks of a head, rounded up
  float eps, inv_d;
  bool interleaved;
};

// A chunk of VEC values, moved as one word of its size (a copy of an array of halves is VEC loads).
template <int BYTES> struct Word;
template <> struct Word<16> { typedef uint4 type; };
template <> struct Word<8> { typedef uint2 type; };
template <> struct Word<4> { typedef uint32_t type; };
template <> struct Word<2> { typedef uint16_t type; };
template <typename T, int VEC>
struct Chunk {
  typedef typename Word<sizeof(T) * VEC>::type W;
  W w;
  __device__ __forceinline__ float get(int i) const { return float(reinterpret_cast<const T*>(&w)[i]); }
  __device__ __forceinline__ void set(int i, float f) { reinterpret_cast<T*>(&w)[i] = T(f); }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < int(sizeof(W) / (sizeof(W) >= 4 ? 4 : 2)); ++i) {
      if (sizeof(W) >= 4) reinterpret_cast<uint32_t*>(&w)[i] = 0u;
      else reinterpret_cast<uint16_t*>(&w)[i] = 0;
    }
  }
  __device__ __forceinline__ float2 pair(int i) const {
    if constexpr (sizeof(T) == 2) return __half22float2(reinterpret_cast<const __half2*>(&w)[i / 2]);
    else return reinterpret_cast<const float2*>(&w)[i / 2];
  }
  __device__ __forceinline__ void set_pair(int i, float2 f) {
    if constexpr (sizeof(T) == 2) reinterpret_cast<__half2*>(&w)[i / 2] = __float22half2_rn(f);
    else reinterpret_cast<float2*>(&w)[i / 2] = f;
  }
  __device__ __forceinline__ void shuffle(int src) {
#pragma unroll
    for (int i = 0; i < int(sizeof(W) / 4); ++i)
      reinterpret_cast<uint32_t*>(&w)[i] = __shfl_sync(0xffffffffu, reinterpret_cast<uint32_t*>(&w)[i], src);
  }
  __device__ __forceinline__ void load(const T* p) { w = *reinterpret_cast<const W*>(p); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<W*>(p) = w; }
};

// N consecutive f32 values, in loads as wide as N allows.
template <int N>
__device__ __forceinline__ void load_f32(float (&f)[N], const float* p) {
  Chunk<float, N> c;
  c.load(p);
#pragma unroll
  for (int i = 0; i < N; ++i) f[i] = c.get(i);
}
template <>
__device__ __forceinline__ void load_f32<8>(float (&f)[8], const float* p) {
  const float4 u = __ldg(reinterpret_cast<const float4*>(p)), v = __ldg(reinterpret_cast<const float4*>(p) + 1);
  f[0] = u.x, f[1] = u.y, f[2] = u.z, f[3] = u.w, f[4] = v.x, f[5] = v.y, f[6] = v.z, f[7] = v.w;
}

// Coefficients of one chunk at values [d, d + VEC): its weights times the cosines and sines. `step`:
// values per angle (1, or 2 when the pairs are neighbours), `angle`: index of the first one.
template <int VEC, int ANGLES>
__device__ __forceinline__ void coefficients(float (&wc)[VEC], float (&ws)[VEC], const float* w, const float* cs, int R,
                                             int d, int angle, bool turned) {
  if (w) {
    load_f32<VEC>(wc, w + d);
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e) wc[e] = 1.f;
  }
#pragma unroll
  for (int e = 0; e < VEC; ++e) ws[e] = 0.f;
  if (turned) {
    float c[ANGLES], s[ANGLES];
    load_f32<ANGLES>(c, cs + angle);
    load_f32<ANGLES>(s, cs + R + angle);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      ws[e] = wc[e] * s[e * ANGLES / VEC];
      wc[e] *= c[e * ANGLES / VEC];
    }
  }
}

// The usual heads (up to 32 chunks): a thread owns one chunk of U heads of a row, so a warp's loads and
// stores are whole heads side by side; the chunk that the rotation mixes with comes from its lane. MODE:
// 0 no rotation, 1 pairs R / 2 apart, 2 neighbouring pairs. Next to the loads it is the instructions that
// count (packed f32x2 arithmetic, one mode to a kernel): 65,536 rows of 24 heads of 64 take 77 us (5.3 TB/s;
// 91 us with every mode in one kernel, 160 instructions to a chunk, and 83 us with the kernel below). Heads
// whose chunks are no power of two (!POW2) share a warp whole: 35,149 rows of 20 heads of 80, 55 us against
// 65 with 16 lanes to their 10 chunks. Four CTAs to an SM for neighbouring pairs, though 64 registers spill 36 bytes
// (20,011 rows of 20 heads of 128, 39 us against 43); pairs R / 2 apart would spill more (99 against 77).
template <typename T, int VEC, int U, int MODE, bool POW2>
__global__ void __launch_bounds__(256, MODE != 2 ? 3 : POW2 ? 4 : 0) qk_norm_rope_lanes_kernel(const NormParams p, int lanes) {
  const int lane = threadIdx.x & 31;
  int c;           // chunk
  uint32_t group;  // blocks of heads, in order
  bool in;         // (all stay for the shuffles)
  if (POW2) {
    const uint32_t log2 = 31 - __clz(lanes);
    group = (blockIdx.x * 256u + threadIdx.x) >> log2;
    c = lane & (lanes - 1);
    in = group < p.groups;
  } else {  // whole heads to a warp, lanes behind the last one idle; lane / lanes is exact below 33
    const uint32_t nth = uint32_t(lane) * p.lane_inv >> 10, of = 32u * p.lane_inv >> 10;
    c = lane - int(nth) * lanes;
    group = (blockIdx.x * 8u + (threadIdx.x >> 5)) * of + nth;
    in = nth < of && group < p.groups;
  }
  const uint32_t row = group / p.blocks, block = group - row * p.blocks;
  const bool is_k = block >= p.q_blocks;
  const int head0 = int(is_k ? block - p.q_blocks : block) * U;
  const int nheads = in ? min(U, (is_k ? p.k_heads : p.q_heads) - head0) : 0;
  const int d = c * VEC;

  int pos = 0;
  if (MODE && in) pos = __ldg(p.positions + row);  // (first: the angles depend on it)
  const int64_t col = int64_t((is_k ? p.q_heads : 0) + head0) * p.D + d;
  const T* xr = static_cast<const T*>(p.x) + row * p.x_stride + col;
  Chunk<T, VEC> a[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    a[u].clear();
    if (u < nheads) a[u].load(xr + u * p.D);
  }
  // y = (x wc + partner's x ws) * scale: ws is the partner's weight times the sine, with its sign
  const float* w = is_k ? p.kw : p.qw;
  float wc[VEC], ws[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) wc[e] = 1.f, ws[e] = 0.f;
  if (in && w) load_f32<VEC>(wc, w + d);
  const int half = p.R / 2 / VEC;  // chunks of half the rotated part
  const bool turned = MODE && in && d < p.R;
  int other = c;
  if constexpr (MODE != 0) {
    if (pos < 0 || pos >= p.table_rows) {  // the row comes out zero
      atomicExch(&kh_norm_error, OP_BAD_INDEX);
      pos = 0;
#pragma unroll
      for (int u = 0; u < U; ++u) a[u].clear();
    }
    const float* cs = p.cossin + int64_t(pos) * 2 * p.R;
    if (MODE == 1 && turned) {
      other = c < half ? c + half : c - half;
      float co[VEC], si[VEC], wo[VEC];
      const int angle = (c < half ? c : other) * VEC;
      load_f32<VEC>(co, cs + angle);
      load_f32<VEC>(si, cs + p.R + angle);
#pragma unroll
      for (int e = 0; e < VEC; ++e) wo[e] = 1.f;
      if (w) load_f32<VEC>(wo, w + other * VEC);
      const float sign = c < half ? -1.f : 1.f;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        ws[e] = sign * wo[e] * si[e];
        wc[e] *= co[e];
      }
    } else if (MODE == 2 && turned) {
      float co[VEC / 2], si[VEC / 2];
      load_f32<VEC / 2>(co, cs + d / 2);
      load_f32<VEC / 2>(si, cs + p.R + d / 2);
#pragma unroll
      for (int e = 0; e < VEC; e += 2) {
        ws[e] = -wc[e + 1] * si[e / 2];
        ws[e + 1] = wc[e] * si[e / 2];
        wc[e] *= co[e / 2];
        wc[e + 1] *= co[e / 2];
      }
    }
  }

  float scale[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float2 ss = make_float2(0.f, 0.f);
#pragma unroll
    for (int e = 0; e < VEC; e += 2) ss = sm100::ffma2(a[u].pair(e), a[u].pair(e), ss);
    scale[u] = ss.x + ss.y;
  }
  if (POW2) {
    for (int o = lanes >> 1; o; o >>= 1)
#pragma unroll
      for (int u = 0; u < U; ++u) scale[u] += __shfl_xor_sync(0xffffffffu, scale[u], o);
  } else {  // towards the head's first lane, and back
    for (int o = 16; o; o >>= 1)
      if (o < lanes)
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const float t = __shfl_down_sync(0xffffffffu, scale[u], o);
          if (c + o < lanes) scale[u] += t;
        }
#pragma unroll
    for (int u = 0; u < U; ++u) scale[u] = __shfl_sync(0xffffffffu, scale[u], lane - c);
  }

  const int src = lane - c + other;
  T* yr = static_cast<T*>(p.out) + row * p.out_stride + col;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const float sc = rsqrtf(fmaf(scale[u], p.inv_d, p.eps));
    Chunk<T, VEC> b = a[u];
    if (MODE == 1) b.shuffle(src);
    // (an unturned value has no partner: 0 times an infinity next to it must not reach it)
    if (MODE && !turned) b.clear();
    if (u >= nheads) continue;
    Chunk<T, VEC> o;
#pragma unroll
    for (int e = 0; e < VEC; e += 2) {
      float2 y = sm100::fmul2(a[u].pair(e), make_float2(wc[e], wc[e + 1]));
      if (MODE) {
        float2 g = b.pair(e);
        if (MODE == 2) g = make_float2(g.y, g.x);
        y = sm100::ffma2(g, make_float2(ws[e], ws[e + 1]), y);
      }
      o.set_pair(e, sm100::fmul2(y, make_float2(sc, sc)));
    }
    o.store(yr + u * p.D);
  }
}

// Heads of more chunks, and unaligned ones: a thread owns chunk i of a head and the one R / 2 values on (neighbours
// where the pairs are neighbours or behind R). LANES threads, a power of two, hold a head. PAIRS: chunk pairs of a thread (1, or 4 for the one-value
// chunks of unaligned heads). LANES * PAIRS pairs cover D <= 256.
template <typename T, int VEC, int PAIRS, int U>
__global__ void __launch_bounds__(256) qk_norm_rope_kernel(const NormParams p, int lanes_log2) {
  const uint32_t lanes = 1u << lanes_log2;
  const uint32_t thread = blockIdx.x * 256u + threadIdx.x;
  const int sub = int(thread & (lanes - 1));
  const uint32_t group = thread >> lanes_log2;
  const uint32_t row = group / p.blocks, block = group - row * p.blocks;
  const bool in = group < p.groups;  // (the threads of a head agree; all stay for the shuffles)
  const bool is_k = block >= p.q_blocks;
  const int head0 = int(is_k ? block - p.q_blocks : block) * U;
  const int nheads = in ? min(U, (is_k ? p.k_heads : p.q_heads) - head0) : 0;
  const int first = (is_k ? p.q_heads : 0) + head0;  // among all heads of the row

  int pos = 0;
  if (in && p.R) pos = p.positions[row];  // (first: the angles depend on it)

  const int chunks = p.D / VEC;
  const int apart = p.interleaved ? 0 : p.R / 2 / VEC;  // pairs whose chunks lie R / 2 values apart
  int c0[PAIRS], c1[PAIRS];
#pragma unroll
  for (int i = 0; i < PAIRS; ++i) {
    const int k = sub + i * int(lanes);
    c0[i] = k < apart ? k : 2 * k;
    c1[i] = k < apart ? k + apart : 2 * k + 1;
    if (c0[i] >= chunks) c0[i] = -1;
    if (c1[i] >= chunks) c1[i] = -1;
  }

  const T* xr = static_cast<const T*>(p.x) + row * p.x_stride + int64_t(first) * p.D;
  Chunk<T, VEC> a[U][PAIRS], b[U][PAIRS];
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) {
      a[u][i].clear();
      b[u][i].clear();
      if (u < nheads) {
        if (c0[i] >= 0) a[u][i].load(xr + u * p.D + c0[i] * VEC);
        if (c1[i] >= 0) b[u][i].load(xr + u * p.D + c1[i] * VEC);
      }
    }

  const bool bad = pos < 0 || (p.R && pos >= p.table_rows);
  if (bad) {
    atomicExch(&kh_norm_error, OP_BAD_INDEX);
    pos = 0;
  }
  const float* cs = p.cossin + int64_t(pos) * 2 * p.R;
  const float* w = is_k ? p.kw : p.qw;

  float scale[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int i = 0; i < PAIRS; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float f = a[u][i].get(e), g = b[u][i].get(e);
        s0 = fmaf(f, f, s0);
        s1 = fmaf(g, g, s1);
      }
    scale[u] = s0 + s1;
  }
  for (uint32_t o = lanes >> 1; o; o >>= 1)
#pragma unroll
    for (int u = 0; u < U; ++u) scale[u] += __shfl_xor_sync(0xffffffffu, scale[u], o);
#pragma unroll
  for (int u = 0; u < U; ++u) scale[u] = bad ? 0.f : rsqrtf(fmaf(scale[u], p.inv_d, p.eps));

  T* yr = static_cast<T*>(p.out) + row * p.out_stride + int64_t(first) * p.D;
#pragma unroll
  for (int i = 0; i < PAIRS; ++i) {
    if (c0[i] < 0 || nheads == 0) continue;
    const int d0 = c0[i] * VEC, d1 = c1[i] * VEC;
    const bool two = c1[i] >= 0, far = sub + i * int(lanes) < apart;
    const bool near0 = p.interleaved && d0 < p.R, near1 = p.interleaved && two && d1 < p.R;
    float wc0[VEC], ws0[VEC], wc1[VEC], ws1[VEC];
    if (p.interleaved) {
      constexpr int N = VEC == 1 ? 1 : VEC / 2;
      coefficients<VEC, N>(wc0, ws0, w, cs, p.R, d0, d0 / 2, near0);
      if (two) coefficients<VEC, N>(wc1, ws1, w, cs, p.R, d1, d1 / 2, near1);
    } else {
      coefficients<VEC, VEC>(wc0, ws0, w, cs, p.R, d0, d0, far);
      if (two) coefficients<VEC, VEC>(wc1, ws1, w, cs, p.R, d1, d0, far);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u >= nheads) break;
      float f[VEC], g[VEC], y0[VEC], y1[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        f[e] = a[u][i].get(e);
        g[e] = b[u][i].get(e);
      }
      // the partner of a value: in the other chunk, or beside it in its own (VEC 1: the other chunk)
      if (far || (VEC == 1 && near0)) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          y0[e] = fmaf(f[e], wc0[e], -(g[e] * ws1[e]));
          y1[e] = fmaf(g[e], wc1[e], f[e] * ws0[e]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          y0[e] = f[e] * wc0[e];
          y1[e] = two ? g[e] * wc1[e] : 0.f;
        }
        if constexpr (VEC > 1) {
          if (near0) {
#pragma unroll
            for (int e = 0; e < VEC; e += 2) {
              y0[e] -= f[e + 1] * ws0[e + 1];
              y0[e + 1] += f[e] * ws0[e];
            }
          }
          if (near1) {
#pragma unroll
            for (int e = 0; e < VEC; e += 2) {
              y1[e] -= g[e + 1] * ws1[e + 1];
              y1[e + 1] += g[e] * ws1[e];
            }
          }
        }
      }
      Chunk<T, VEC> o;
#pragma unroll
      for (int e = 0; e < VEC; ++e) o.set(e, bad ? 0.f : y0[e] * scale[u]);
      o.store(yr + u * p.D + d0);
      if (two) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) o.set(e, bad ? 0.f : y1[e] * scale[u]);
        o.store(yr + u * p.D + d1);
      }
    }
  }
}

// PAIRS 0: the kernel with one chunk to a thread.
template <typename T, int VEC, int PAIRS, int U>
void launch(NormParams p, int64_t rows, cudaStream_t st) {
  int log2 = 0;
  while ((std::max(PAIRS, 1) << log2) < (p.D / VEC + 1) / 2) ++log2;
  const int lanes = p.D / VEC, heads = PAIRS ? 32 >> log2 : 32 / lanes;  // heads (of U blocks) of a warp
  p.q_blocks = uint32_t((p.q_heads + U - 1) / U);
  p.blocks = p.q_blocks + uint32_t((p.k_heads + U - 1) / U);
  p.lane_inv = uint32_t((1024 + lanes - 1) / lanes);
  // 32-bit thread indexes: launches of as many whole rows as stay below 2^31 threads
  const int64_t most = ((int64_t(1) << 31) - 8192) / 32 * heads / p.blocks;
  for (int64_t r = 0; r < rows; r += most) {
    const int64_t n = std::min(most, rows - r);
    NormParams q = p;
    q.groups = uint32_t(n * p.blocks);
    q.x = static_cast<const T*>(p.x) + r * p.x_stride;
    q.out = static_cast<T*>(p.out) + r * p.out_stride;
    if (p.R) q.positions = p.positions + r;
    const unsigned grid = unsigned((q.groups + 8 * heads - 1) / (8 * heads));
    if constexpr (PAIRS == 0) {
      const int mode = !p.R ? 0 : !p.interleaved ? 1 : 2;
      auto go = [&](auto* kernel) { kernel<<<grid, 256, 0, st>>>(q, lanes); };
      if ((lanes & (lanes - 1)) == 0)
        go(mode == 0 ? qk_norm_rope_lanes_kernel<T, VEC, U, 0, true> : mode == 1 ? qk_norm_rope_lanes_kernel<T, VEC, U, 1, true>
                                                                                 : qk_norm_rope_lanes_kernel<T, VEC, U, 2, true>);
      else
        go(mode == 0 ? qk_norm_rope_lanes_kernel<T, VEC, U, 0, false> : mode == 1 ? qk_norm_rope_lanes_kernel<T, VEC, U, 1, false>
                                                                                  : qk_norm_rope_lanes_kernel<T, VEC, U, 2, false>);
    } else {
      qk_norm_rope_kernel<T, VEC, PAIRS, U><<<grid, 256, 0, st>>>(q, log2);
    }
  }
  KH_CUDA(cudaGetLastError());
}

// Whether chunks of `vec` values fit the head, its rotation and the alignment of rows, angles, weights.
bool fits(const kh_qk_norm_rope_args& a, int size, int vec) {
  const uintptr_t bytes = uintptr_t(vec) * size;
  auto at = [](const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; };
  return a.head_dim % vec == 0 && (a.interleaved ? a.rotary_dim : a.rotary_dim / 2) % vec == 0 && at(a.x, bytes) &&
         at(a.out, bytes) && a.x_stride % vec == 0 && a.out_stride % vec == 0 && at(a.q_weight, 16) &&
         at(a.k_weight, 16) && (a.rotary_dim == 0 || at(a.cossin, 16)) && a.rotary_dim % 4 == 0;
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
  check_that(a.rows >= 0 && a.rows < (int64_t(1) << 31), fn, "rows must be in [0, 2^31)");
  const int64_t width = int64_t(a.q_heads + a.k_heads) * a.head_dim;
  check_that(a.x_stride >= width && a.out_stride >= width && a.x_stride < (int64_t(1) << 31) &&
                 a.out_stride < (int64_t(1) << 31),
             fn, "strides must be at least (q_heads + k_heads) * head_dim and below 2^31");
  check_that(a.rows * std::max(a.x_stride, a.out_stride) < (int64_t(1) << 48), fn, "rows * stride must be below 2^48");
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
    check_that(aligned4(a.cossin) && aligned4(a.positions), fn, "cossin and positions must be 4-byte aligned");
  }
  check_that(aligned4(a.q_weight) && aligned4(a.k_weight), fn, "weights must be 4-byte aligned");
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
    if (fits(a, 2, 8)) launch<__half, 8, 0, 4>(p, a.rows, st);
    else if (fits(a, 2, 4) && a.head_dim <= 128) launch<__half, 4, 0, 4>(p, a.rows, st);
    else launch<__half, 1, 4, 1>(p, a.rows, st);
  } else {
    if (fits(a, 4, 4) && a.head_dim <= 128) launch<float, 4, 0, 4>(p, a.rows, st);
    else if (fits(a, 4, 4)) launch<float, 4, 1, 2>(p, a.rows, st);
    else launch<float, 1, 4, 1>(p, a.rows, st);
  }
}

int* qk_norm_index_word() {
  void* p = nullptr;
  KH_CUDA(cudaGetSymbolAddress(&p, kh_norm_error));
  return static_cast<int*>(p);
}

}  // namespace kh
