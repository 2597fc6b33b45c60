// A projection with the low-rank adapters of many requests.
//
// out[t] = x[t] W^T + bias + s_a (x[t] A_a^T) B_a^T, a the adapter of the segment of rows that t lies
// in. Two launches: h[t] = s_a x[t] A_a^T (rank values a row, rounded to f16: 2^-11 of the adapter's
// own part; rows with a value beyond f16: see row_beyond_f16), then the projection with h B_a^T added to
// the same f32 accumulators, rounded once. The second launch starts while the first runs (programmatic
// dependent launch) and waits for it where it needs h, behind the projection's own products. (One launch
// where few rows have few adapters: see lora_few_kernel.)
//
// Few rows (takes_few): bound by reading W, A and B once; lora_shrink_rows_kernel and
// lora_few_kernel. Many rows: bound by the tensor cores;
// lora_shrink_tile_kernel (HBM: reads x once) and lora_pair_kernel. A row tile that holds rows of
// several adapters takes one more product per adapter, whose output lanes of other rows are switched
// off in the instruction, so no operand is masked or copied, and rows of one adapter need not be neighbours.
// (h is made with one product an adapter and tile; the projection lists a tile's adapters from 32 segments at a
// time, so one that comes back in later segments takes a product again: 1,000 single rows of 60 adapters take
// 233 to a tile of 256 rows.)
// Times beside the kernels and rules are of calls in a graph, unless a single launch is named; calls queued one by
// one from a program take 1 to 2 us more.

#include "device_ops.h"

#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <cmath>

#include "runtime.h"
#include "sm100.cuh"
#include "tmap.h"

namespace kh {

namespace {

using namespace sm100;

__device__ int kh_lora_index_error = 0;  // (a wait that gave up: kh_tc_error)

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
  __half* h;  // [rows][rank]
  int64_t rows, x_stride, out_stride;
  int k, n, rank, n_adapters, n_segs;
};

// Start of segment i, cut to the buffer.
__device__ __forceinline__ int seg_start(const LoraParams& p, int i) {
  return int(min(max(int64_t(__ldg(p.starts + i)), int64_t(0)), p.rows));
}
// An id as an adapter, -1 for none; one that does not exist counts as none and is reported.
__device__ __forceinline__ int known_adapter(const LoraParams& p, int id) {
  if (id < p.n_adapters) return id < 0 ? -1 : id;
  atomicOr(&kh_lora_index_error, OP_BAD_INDEX);
  return -1;
}
__device__ __forceinline__ int adapter_of(const LoraParams& p, int seg) { return known_adapter(p, __ldg(p.ids + seg)); }
// First segment that ends behind row r (n_segs if none), found by a whole warp, 32 probes a round; with one
// row to a segment (a step of single tokens) it is segment r, which the first round looks at too. Where the
// caller's first round reads all segments anyway (`reads` of them), the first of all.
__device__ __forceinline__ int first_seg(const LoraParams& p, int r, int reads) {
  if (p.n_segs <= reads) return 0;
  const int lane = threadIdx.x & 31;
  const int guess = min(r, p.n_segs - 1), g0 = seg_start(p, guess), g1 = seg_start(p, guess + 1);
  int lo = 0, hi = p.n_segs;
  while (lo < hi) {
    const int step = (hi - lo + 31) / 32, i = lo + lane * step;
    const uint32_t ended = __ballot_sync(0xffffffffu, i < hi && seg_start(p, i + 1) <= r);
    if (g0 <= r && r < g1) return guess;
    const int c = ended == 0xffffffffu ? 32 : __ffs(~ended) - 1;  // probes before the first that has not
    if (c == 0) return lo;
    hi = min(hi, lo + c * step);
    lo += (c - 1) * step + 1;
  }
  return lo;
}

__device__ __forceinline__ float dot8(uint4 a, uint4 b, float acc) {
  const __half2* x = reinterpret_cast<const __half2*>(&a);
  const __half2* y = reinterpret_cast<const __half2*>(&b);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 u = __half22float2(x[i]), v = __half22float2(y[i]);
    acc = fmaf(u.x, v.x, fmaf(u.y, v.y, acc));
  }
  return acc;
}

// Dot product of k values by a whole warp, the same in every lane.
__device__ __forceinline__ float warp_dot(const __half* x, const __half* y, int k) {
  const uint4 *u = reinterpret_cast<const uint4*>(x), *v = reinterpret_cast<const uint4*>(y);
  float d = 0.f;
#pragma unroll 1
  for (int i = threadIdx.x & 31; i < k / 8; i += 32) d = dot8(__ldg(u + i), __ldg(v + i), d);
  for (int o = 16; o; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
  return d;
}
// h is an f16 operand, so a value of it beyond 65,504 is an infinity, and all that it is multiplied with is
// infinite or NaN. A row with such outputs comes here, to one warp: its h in f32, and where a value may have
// been too large (2^15: this sum's order is another one) `count` outputs from n0 on again, put(j, value) by every
// lane. Otherwise the row is infinite by the definition, and stays as it is.
template <class Put>
__device__ __forceinline__ void row_beyond_f16(const LoraParams& p, int64_t row, int ad, int n0, int count, Put put) {
  const int lane = threadIdx.x & 31;
  const __half* x = p.x + row * p.x_stride;
  const float s = p.scales ? __ldg(p.scales + ad) : 1.f;
  float h[4] = {};  // rank value lane + 32 i
  bool beyond = false;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll 1
    for (int r = 32 * i; r < min(32 * i + 32, p.rank); ++r) {
      const float d = warp_dot(x, p.a + (int64_t(ad) * p.rank + r) * p.k, p.k) * s;
      if (lane == (r & 31)) h[i] = d;
      beyond |= fabsf(d) >= 32768.f && fabsf(d) < INFINITY;
    }
  if (!beyond) return;
#pragma unroll 1
  for (int j = 0; j < count; ++j) {
    const int n = n0 + j;
    const __half* b = p.b + (int64_t(ad) * p.n + n) * p.rank;
    float d = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (lane + 32 * i < p.rank) d = fmaf(h[i], __half2float(b[lane + 32 * i]), d);
    for (int o = 16; o; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
    put(j, warp_dot(x, p.w + int64_t(n) * p.k, p.k) + d + (p.bias ? __half2float(p.bias[n]) : 0.f));
  }
}

// ---- few rows: h, one CTA of 16 warps per row, a warp one of the rank's dot products at a time ----

__global__ void __launch_bounds__(512) lora_shrink_rows_kernel(const LoraParams p) {
  launch_dependents();
  const int t = blockIdx.x, lane = threadIdx.x & 31;
  const int seg = first_seg(p, t, 0);
  if (seg >= p.n_segs || t < seg_start(p, seg) || t >= seg_start(p, p.n_segs)) return;
  const int ad = adapter_of(p, seg);
  if (ad < 0) return;
  const uint4* x = reinterpret_cast<const uint4*>(p.x + t * p.x_stride);
  const float s = p.scales ? __ldg(p.scales + ad) : 1.f;
  const int chunks = p.k / 8;
  for (int r = threadIdx.x >> 5; r < p.rank; r += 16) {
    const uint4* a = reinterpret_cast<const uint4*>(p.a + (int64_t(ad) * p.rank + r) * p.k);
    float d = 0.f;
    int i = lane;
    for (; i + 7 * 32 < chunks; i += 8 * 32) {  // eight loads of each in flight
      uint4 u[8], v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        u[j] = __ldg(a + i + 32 * j);
        v[j] = __ldg(x + i + 32 * j);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) d = dot8(u[j], v[j], d);
    }
#pragma unroll 4
    for (; i < chunks; i += 32) d = dot8(__ldg(a + i), __ldg(x + i), d);
    for (int o = 16; o; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
    if (lane == 0) p.h[int64_t(t) * p.rank + r] = __float2half_rn(d * s);
  }
}

// ---- few rows: the projection ----
//
// out^T = W x^T: the 128 rows of the MMA are outputs and its columns the (up to 128) rows of x, so that
// few rows waste no tensor work and W streams once through a deep ring. A cluster of Z CTAs splits the
// sum of 128 outputs, until about every SM takes part in reading W, and adds the parts over distributed
// shared memory in rank order, each CTA for its share of the rows, in groups of eight. The adapters' part
// of a group is m16n8k16 products of B's rows as they lie in memory with the group's h, one adapter's rows
// of it at a time (as dot products, a thread to an output, 120 rows of 4 adapters of rank 64, 4,096 ->
// 4,096, took 49 us; so, 36). Warp 0 TMA, warp 1 MMA, warps 2-9 16 outputs each, warp 10 finds the rows'
// adapters meanwhile.
// FUSED: where all adapters' A together have at most 128 rows, they are a second operand tile of every
// stage, h comes out of the same pass over x, and there is no launch before this one.
// 64 rows of 48 adapters of rank 16, 4,096 -> 4,096: 19.2 us, of it 2.6 to the first tile, 4 to 6 for W (46 MB
// with the adapters), 5 for the sum, the adapters and the outputs.

constexpr int FT = 128;      // rows of x, at most
constexpr int FTHREADS = 352;
constexpr int FSMEM = 200 * 1024;

__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

constexpr int PS = 132;  // row stride of the parts of the sum: [row of x][output], f32

// The adapters' part: products of B's rows, 16 outputs to a warp, with the h of eight rows of x, one
// adapter's rows of them at a time (zeros for the others). A CTA's products go through its groups of rows,
// a group's adapters and the rank's sixteens, eight of one group to a batch, whose loads of B are in flight
// together: those of the first from before the sum is done, the others' under the products before them.
// The order of the rank's values is free: the quad lane q takes the values 4 q .. 4 q + 3 of 16, of B and h.
struct Products {
  int g;             // group
  int mine;          // adapter of the row of x that this lane holds h of
  uint32_t leaders;  // a lane for each adapter that is left
  int k;             // first of the adapter's rank values that are left
  // the next group with an adapter, from g on
  __device__ __forceinline__ void find(const int* ids, int nt, int step) {
    const int lane = threadIdx.x & 31;
    for (; g * 8 < nt; g += step) {
      mine = ids[g * 8 + (lane >> 2)];
      const uint32_t same = __match_any_sync(0xffffffffu, mine);
      leaders = __ballot_sync(0xffffffffu, mine >= 0 && lane == __ffs(same) - 1);
      if (leaders) return;
    }
  }
  __device__ __forceinline__ int adapter() const { return __shfl_sync(0xffffffffu, mine, __ffs(leaders) - 1); }
  __device__ __forceinline__ void next(int rank) {
    k += 16;
    if (k >= rank) {
      k = 0;
      leaders &= leaders - 1;
    }
  }
};
// b: B at this lane's output and rank values, of adapter 0; low, high: its outputs lane / 4 and + 8 exist
__device__ __forceinline__ void load_batch(const LoraParams& p, Products& s, const int* ids, int nt, int step, const __half* b,
                                           bool low, bool high, uint2 (&lo)[8], uint2 (&hi)[8]) {
  const int q4 = (threadIdx.x & 3) * 4;
  const uint32_t stride = uint32_t(p.n) * uint32_t(p.rank);  // below 2^23
#pragma unroll
  for (int i = 0; i < 8; ++i) lo[i] = hi[i] = make_uint2(0, 0);
  if (s.g * 8 >= nt) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (s.leaders) {
      const __half* src = b + uint64_t(uint32_t(s.adapter())) * stride + s.k;
      if (s.k + q4 < p.rank) {
        if (low) lo[i] = __ldg(reinterpret_cast<const uint2*>(src));
        if (high) hi[i] = __ldg(reinterpret_cast<const uint2*>(src + 8 * p.rank));
      }
      s.next(p.rank);
    }
  }
  if (!s.leaders) {
    s.g += step;
    s.find(ids, nt, step);
  }
}
// part: the sum at row 0 of x and this lane's output; hs: h [row of x][rank + 8]. A product is taken over in the
// columns of its own adapter's rows alone: the zeros that stand for the other rows' h would turn an infinity
// in this adapter's B into a NaN in their outputs.
__device__ __forceinline__ void use_batch(const LoraParams& p, Products s, const __half* hs, float* part, const uint2 (&lo)[8],
                                          const uint2 (&hi)[8]) {
  const int lane = threadIdx.x & 31, q4 = (lane & 3) * 4;
  float* dst = part + (s.g * 8 + 2 * (lane & 3)) * PS;
  float acc[4] = {dst[0], dst[PS], dst[8], dst[PS + 8]};
  const int column0 = __shfl_sync(0xffffffffu, s.mine, 8 * (lane & 3)), column1 = __shfl_sync(0xffffffffu, s.mine, 8 * (lane & 3) + 4);
  const __half* h = hs + (s.g * 8 + (lane >> 2)) * (p.rank + 8) + q4;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (!s.leaders) break;
    const int id = s.adapter();
    uint2 v = make_uint2(0, 0);
    if (id == s.mine && s.k + q4 < p.rank) v = *reinterpret_cast<const uint2*>(h + s.k);
    s.next(p.rank);
    float sum[4] = {acc[0], acc[1], acc[2], acc[3]};
    mma_16816(sum, lo[i].x, hi[i].x, lo[i].y, hi[i].y, v.x, v.y);
    if (id == column0) acc[0] = sum[0], acc[2] = sum[2];
    if (id == column1) acc[1] = sum[1], acc[3] = sum[3];
  }
  dst[0] = acc[0];
  dst[PS] = acc[1];
  dst[8] = acc[2];
  dst[PS + 8] = acc[3];
}

// cols: rows of x rounded up to the MMA's steps of 16; a stage: 16 KB of W, FUSED 16 KB of A (of them
// a_bytes loaded), cols * 128 bytes of x.
// (registers: what leaves an SM room for a CTA of lora_shrink_rows_kernel)
template <bool FUSED>
__global__ void __maxnreg__(FUSED ? 168 : 112)
    lora_few_kernel(const __grid_constant__ CUtensorMap tmx, const __grid_constant__ CUtensorMap tmw,
                    const __grid_constant__ CUtensorMap tma, const LoraParams p, int Z, int cols, int stages, int a_bytes) {
  constexpr int X_OFF = FUSED ? 32768 : 16384;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t bars[2 * 12 + 2];
  __shared__ uint32_t tmem_holder;
  __shared__ volatile int abort_flag;
  __shared__ int ids[FT];
  __shared__ float row_scale[FT];  // (FUSED)
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int z = blockIdx.x % Z, n0 = int(blockIdx.x / Z) * 128;
  const int begin = seg_start(p, 0), end = seg_start(p, p.n_segs);
  const int t0 = begin + int(blockIdx.y) * FT;
  if (t0 >= end) {  // (the whole cluster)
    wait_primary();
    return;
  }
  const int nt = min(FT, end - t0);
  const int x_bytes = cols * 128, stage_bytes = X_OFF + x_bytes;
  uint64_t *full = bars, *empty = bars + stages, *done = bars + 24, *drain = bars + 25;
  const uint32_t tcols = (cols <= 32 ? 32u : cols <= 64 ? 64u : 128u) * (FUSED ? 2 : 1);
  if (threadIdx.x == 0) {
    for (int i = 0; i < stages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(done, 1);
    mbar_init(drain, 1);
    abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) tmem_alloc(&tmem_holder, tcols);
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  const uint32_t tmem = tmem_holder;
  const int nk_all = (p.k + 63) / 64, kps = (nk_all + Z - 1) / Z;
  const int kb0 = min(z * kps, nk_all), nk = min(kps, nk_all - kb0);
  auto wwait = [&](uint64_t* bar, uint32_t parity, int code) -> bool {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, code));
  };
  // (warps 2-9)
  Products loaded, used;
  uint2 b_lo[8], b_hi[8];
  const int m = n0 + 16 * (warp - 2) + (lane >> 2);  // output of this lane's rows of B
  const bool low = m < p.n, high = m + 8 < p.n;
  const __half* b_at = p.b + int64_t(m) * p.rank + (lane & 3) * 4;

  if (warp == 0) {
    bool ok = true;
    int st = 0;
    uint32_t ph = 0, pend = 0;
    for (int kb = 0; kb < nk; ++kb) {
      if (!wwait(&empty[st], ph ^ 1, 231)) { ok = false; break; }
      if (lane == 0) {
        mbar_arrive_expect_tx(&full[st], uint32_t(16384 + x_bytes + (FUSED ? a_bytes : 0)));
        tma_load_2d(smem + st * stage_bytes, &tmw, &full[st], (kb0 + kb) * 64, n0);
        if (FUSED) tma_load_2d(smem + st * stage_bytes + 16384, &tma, &full[st], (kb0 + kb) * 64, 0);
        tma_load_2d(smem + st * stage_bytes + X_OFF, &tmx, &full[st], (kb0 + kb) * 64, t0);
      }
      __syncwarp();
      pend = (pend & ~(3u << (2 * st))) | ((2u | ph) << (2 * st));
      if (++st == stages) {
        st = 0;
        ph ^= 1;
      }
    }
    if (!ok) {
      abort_flag = 1;
      for (int i = 0; i < stages; ++i)
        if ((pend >> (2 * i)) & 2u) mbar_wait(&full[i], (pend >> (2 * i)) & 1u, 232);
    }
  } else if (warp == 1) {
    // all lanes in step, one issues
    const uint32_t idesc = idesc_f16(128, cols);
    const bool lead = elect_one();
    bool ok = true;
    int st = 0;
    uint32_t ph = 0;
    for (int kb = 0; kb < nk; ++kb) {
      if (!wwait(&full[st], ph, 233)) { ok = false; break; }
      fence_after_sync();
      const uint64_t dw = desc_sw128(smem + st * stage_bytes), dx = desc_sw128(smem + st * stage_bytes + X_OFF);
#pragma unroll
      for (int k = 0; k < 4; ++k) mma_f16_if(lead, tmem, dw + uint64_t(2 * k), dx + uint64_t(2 * k), idesc, (kb | k) ? 1u : 0u);
      if (FUSED) {  // (rows of the A tile past the adapters hold anything; so do their lanes)
        const uint64_t da = desc_sw128(smem + st * stage_bytes + 16384);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          mma_f16_if(lead, tmem + tcols / 2, da + uint64_t(2 * k), dx + uint64_t(2 * k), idesc, (kb | k) ? 1u : 0u);
      }
      mma_commit_if(lead, &empty[st]);
      __syncwarp();
      if (++st == stages) {
        st = 0;
        ph ^= 1;
      }
    }
    if (!ok) {
      abort_flag = 1;
      if (lead) mma_commit(drain);
      __syncwarp();
      mbar_wait(drain, 0, 234);
    }
    if (lead) mma_commit(done);  // (after a failure too: nothing is stored then)
    __syncwarp();
  } else if (warp == 10) {
    for (int t = lane; t < FT; t += 32) ids[t] = -1;
    __syncwarp();
    for (int s = first_seg(p, t0, 128), more = 1; more && s < p.n_segs; s += 128) {
      // four segments a lane, their loads together
      int lo[4], hi[4], id[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = s + 32 * j + lane;
        lo[j] = hi[j] = t0 + nt;
        id[j] = -1;
        if (i < p.n_segs) {
          lo[j] = max(seg_start(p, i), t0);
          hi[j] = min(seg_start(p, i + 1), t0 + nt);
          id[j] = __ldg(p.ids + i);
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (lo[j] < hi[j]) {
          const int ad = known_adapter(p, id[j]);
          const float sc = FUSED && ad >= 0 && p.scales ? __ldg(p.scales + ad) : 1.f;
          for (int t = lo[j]; t < hi[j]; ++t) {
            ids[t - t0] = ad;
            if (FUSED) row_scale[t - t0] = sc;
          }
        }
      more = __all_sync(0xffffffffu, lo[3] < t0 + nt);
    }
    __syncwarp();
    named_bar(1, 32 * 9);
  } else {
    named_bar(1, 32 * 9);
    loaded.g = z;
    loaded.k = 0;
    loaded.find(ids, nt, Z);
    used = loaded;
    load_batch(p, loaded, ids, nt, Z, b_at, low, high, b_lo, b_hi);
    // the accumulator (lane = output, column = row of x) as part[row of x][output], over the stages,
    // which all have been read
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    const bool ok = wwait(done, 0, 235);
    fence_after_sync();
    float* part = reinterpret_cast<float*>(smem) + quarter * 32 + lane;
    const uint32_t taddr = tmem + (uint32_t(quarter * 32) << 16);
    if (!ok) abort_flag = 1;
#pragma unroll 1
    for (int c = 16 * half; c < cols; c += 32) {
      uint32_t v[16];
      tmem_ld16(taddr + uint32_t(c), v);
      tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        asm volatile("" : "+r"(v[i]));
        part[(c + i) * PS] = nk > 0 ? __uint_as_float(v[i]) : 0.f;
      }
      if (FUSED) {  // the adapters' lanes behind it
        tmem_ld16(taddr + tcols / 2 + uint32_t(c), v);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          asm volatile("" : "+r"(v[i]));
          part[(cols + c + i) * PS] = nk > 0 ? __uint_as_float(v[i]) : 0.f;
        }
      }
    }
  }
  fence_before_sync();
  __syncthreads();
  // outputs that this lane stores, and their bias
  const int n = n0 + 4 * lane;
  uint2 bias_bits = make_uint2(0, 0);
  if (p.bias && n < p.n) bias_bits = __ldg(reinterpret_cast<const uint2*>(p.bias + n));
  if (Z > 1) cluster_sync();
  float* part = reinterpret_cast<float*>(smem);
  // h of this CTA's rows of x, in shared memory, a warp per row
  __half* hs = reinterpret_cast<__half*>(part + (FUSED ? 2 : 1) * cols * PS);  // [row of x][rank + 8]
  if (!FUSED) wait_primary();
  if (p.n_adapters > 0) {
    for (int k = warp; k < FT; k += FTHREADS / 32) {
      const int i = (k / 8 * Z + z) * 8 + k % 8;  // k-th row of this CTA's groups
      if (i >= nt) break;
      const int ad = ids[i];
      if (ad < 0) continue;
      if (FUSED) {  // the parts of the row's own adapter, scaled
        const float sc = row_scale[i];
        for (int r = lane; r < p.rank; r += 32) {
          const float* src = part + (cols + i) * PS + ad * p.rank + r;
          float d = 0.f;
          if (Z == 1) {
            d = *src;
          } else {
            float u[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) u[q] = q < Z ? ld_cluster_f32(cluster_addr(src, uint32_t(q))) : 0.f;
#pragma unroll
            for (int q = 0; q < 8; ++q) d += u[q];
          }
          hs[i * (p.rank + 8) + r] = __float2half_rn(d * sc);
        }
      } else if (lane < p.rank / 8) {
        reinterpret_cast<uint4*>(hs + i * (p.rank + 8))[lane] = reinterpret_cast<const uint4*>(p.h + int64_t(t0 + i) * p.rank)[lane];
      }
    }
    __syncthreads();
    if (warp >= 2 && warp < 10)
      while (used.g * 8 < nt) {
        const Products after = loaded;
        uint2 lo[8], hi[8];
        load_batch(p, loaded, ids, nt, Z, b_at, low, high, lo, hi);
        use_batch(p, used, hs, part + 16 * (warp - 2) + (lane >> 2), b_lo, b_hi);
        used = after;
#pragma unroll
        for (int i = 0; i < 8; ++i) b_lo[i] = lo[i], b_hi[i] = hi[i];
      }
    __syncthreads();
  }
  // this CTA's rows, a warp a row: the parts of the sum, in rank order, and the bias, rounded once
  uint32_t not_finite = 0;  // rows of this warp with an output of this lane that is infinite or NaN
  if (n < p.n && !abort_flag) {
    const float2 bias_lo = __half22float2(*reinterpret_cast<const __half2*>(&bias_bits.x));
    const float2 bias_hi = __half22float2(*reinterpret_cast<const __half2*>(&bias_bits.y));
    const float4 bias = make_float4(bias_lo.x, bias_lo.y, bias_hi.x, bias_hi.y);
#pragma unroll 2
    for (int j = 0; warp + j * (FTHREADS / 32) < FT; ++j) {
      const int k = warp + j * (FTHREADS / 32), i = (k / 8 * Z + z) * 8 + k % 8;
      if (i >= nt) break;
      const float* src = part + i * PS + 4 * lane;
      float4 v = bias;
      float4 u[8];
#pragma unroll
      for (int q = 0; q < 8; ++q)
        u[q] = q >= Z ? make_float4(0.f, 0.f, 0.f, 0.f) : Z == 1 ? *reinterpret_cast<const float4*>(src) : ld_cluster_f32x4(cluster_addr(src, uint32_t(q)));
#pragma unroll
      for (int q = 0; q < 8; ++q) v.x += u[q].x, v.y += u[q].y, v.z += u[q].z, v.w += u[q].w;
      *reinterpret_cast<uint2*>(p.out + (t0 + i) * p.out_stride + n) = make_uint2(pack_half2(v.x, v.y), pack_half2(v.z, v.w));
      const float zero = fmaf(v.x, 0.f, fmaf(v.y, 0.f, fmaf(v.z, 0.f, v.w * 0.f)));
      if (zero != 0.f) not_finite |= 1u << j;
    }
  }
  __syncwarp();  // (such a row is written again, over what other lanes wrote)
  for (not_finite = __reduce_or_sync(0xffffffffu, not_finite); not_finite; not_finite &= not_finite - 1) {
    const int k = warp + (__ffs(not_finite) - 1) * (FTHREADS / 32), i = (k / 8 * Z + z) * 8 + k % 8;
    if (ids[i] < 0) continue;
    __half* dst = p.out + (t0 + i) * p.out_stride + n0;
    row_beyond_f16(p, t0 + i, ids[i], n0, min(128, p.n - n0), [&](int j, float v) {
      if (lane == 0) dst[j] = __float2half_rn(v);
    });
  }
  if (Z > 1) cluster_sync();  // no CTA leaves while another reads its part
  if (warp == 1) {
    fence_after_sync();
    tmem_free(tmem, tcols);
  }
}

// ---- many rows: h on the tensor cores ----
//
// One cluster of Z CTAs per 128 rows, the CTAs splitting the sum (launches of few tiles; while SMs are idle
// then, the tile's adapters are dealt to several clusters too). A K block of
// 64: one tile of x, then for every adapter of the tile's rows its block of A (rank rows) and the
// products, whose lanes of other rows are off, into one accumulator of 128 x rank. 224 threads:
// warp 0 loads x (TMA), warp 1 issues the products, warps 2-5 write the scaled f16 rows, warp 6 finds
// the adapters of the rows, while x loads, and then loads A. (One warp for both loads was the bound: a
// stage costs its issuing thread some 500 cycles.)

constexpr int SXS = 4;  // x stages
constexpr int SAS = 8;  // A stages, at most
constexpr int LISTED = 128;  // adapters of a tile, at most: its rows
struct ShrinkPieces {  // the adapters of a tile
  int count;
  int id[LISTED];
  uint4 off[LISTED];      // lanes of other rows
  int row_id[128];        // adapter of each row, -1 for none (from the warps that write h)
  float row_scale[128];
};

__device__ __forceinline__ uint32_t lanes_on(int lo, int hi, int word) {
  const int a = min(max(lo - 32 * word, 0), 32), b = min(max(hi - 32 * word, 0), 32);
  const uint32_t ub = b >= 32 ? 0xffffffffu : (1u << b) - 1u, ua = a >= 32 ? 0xffffffffu : (1u << a) - 1u;
  return ub & ~ua;
}

__global__ void __launch_bounds__(224) lora_shrink_tile_kernel(const __grid_constant__ CUtensorMap tmx,
                                                               const __grid_constant__ CUtensorMap tma,
                                                               const LoraParams p, int Z, int groups, int xstages,
                                                               int astages) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ ShrinkPieces pieces;
  __shared__ uint64_t bars[2 * SXS + 2 * SAS + 3];
  __shared__ uint32_t tmem_holder;
  __shared__ volatile int abort_flag;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int R16 = (p.rank + 15) / 16 * 16;
  const int a_bytes = R16 * 128;
  uint8_t* sX = smem;
  uint8_t* sA = smem + xstages * 16384;
  uint64_t *x_full = bars, *x_empty = x_full + SXS, *a_full = x_empty + SXS, *a_empty = a_full + SAS,
           *done = a_empty + SAS, *drain = done + 1, *listed = drain + 1;
  launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) prefetch_tmap(&tmx);
  if (threadIdx.x == 192) prefetch_tmap(&tma);
  const int z = blockIdx.x % Z, r0 = int(blockIdx.x / Z) * 128;
  const uint32_t cols = R16 <= 32 ? 32u : R16 <= 64 ? 64u : 128u;
  if (threadIdx.x == 0) {
    for (int i = 0; i < SXS; ++i) {
      mbar_init(&x_full[i], 1);
      mbar_init(&x_empty[i], 1);
    }
    for (int i = 0; i < SAS; ++i) {
      mbar_init(&a_full[i], 1);
      mbar_init(&a_empty[i], 1);
    }
    mbar_init(done, 1);
    mbar_init(drain, 1);
    mbar_init(listed, 32);
    abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) tmem_alloc(&tmem_holder, cols);
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  const uint32_t tmem = tmem_holder;
  const int nk_all = (p.k + 63) / 64, kps = (nk_all + Z - 1) / Z;
  const int kb0 = min(z * kps, nk_all), nk = min(kps, nk_all - kb0);
  auto wwait = [&](uint64_t* bar, uint32_t parity, int code) -> bool {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, code));
  };

  if (warp == 0) {  // all lanes in step, one issues (and so below)
    const bool lead = elect_one();
    bool ok = true;
    int xs = 0, issued = 0;
    uint32_t u = 0;
    for (int kb = 0; kb < nk; ++kb) {
      // past the first round it is known whether any row has an adapter (if none, x was loaded in vain)
      if (kb == xstages && (!wwait(listed, 0, 200) || pieces.count == 0)) break;
      if (!wwait(&x_empty[xs], u ^ 1, 201)) { ok = false; break; }
      mbar_arrive_expect_tx_if(lead, &x_full[xs], 16384);
      tma_load_2d_if(lead, sX + xs * 16384, &tmx, &x_full[xs], (kb0 + kb) * 64, r0);
      __syncwarp();
      ++issued;
      if (++xs == xstages) {
        xs = 0;
        u ^= 1;
      }
    }
    // every copy lands before the CTA ends, also where no product waits for it
    for (int kb = max(issued - xstages, 0); kb < issued; ++kb)
      mbar_wait(&x_full[kb % xstages], uint32_t(kb / xstages) & 1, 203);
    if (!ok) abort_flag = 1;
  } else if (warp == 6) {
    // the adapters of these rows, each with all its rows
    const int last = seg_start(p, p.n_segs);  // rows from here on are not written
    int n = 0;
    for (int s = first_seg(p, r0, 128), more = 1; more && s < p.n_segs; s += 128) {
      // four segments a lane, their loads together
      int lo[4], hi[4], id[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = s + 32 * j + lane;
        lo[j] = hi[j] = 128;
        id[j] = -1;
        if (i < p.n_segs) {
          lo[j] = max(seg_start(p, i), r0) - r0;
          hi[j] = min(min(seg_start(p, i + 1), last), r0 + 128) - r0;
          id[j] = __ldg(p.ids + i);
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (!__any_sync(0xffffffffu, lo[j] < hi[j])) continue;
        int ad = lo[j] < hi[j] ? known_adapter(p, id[j]) : -1;
        if (ad % groups != int(blockIdx.y)) ad = -1;  // (-1 % groups is no group's)
        // an adapter that is in the list already takes these rows too; a new one's first lane adds it
        int at = -1;
        for (int k = 0; k < n; ++k) at = pieces.id[k] == ad ? k : at;
        const uint32_t peers = __match_any_sync(0xffffffffu, ad);
        const bool fresh = ad >= 0 && at < 0;
        const uint32_t added = __ballot_sync(0xffffffffu, fresh && lane == __ffs(peers) - 1);
        if (fresh) at = n + __popc(added & ((1u << (__ffs(peers) - 1)) - 1u));
        if (at >= LISTED) {  // only where starts decrease: else every adapter has a row of its own
          atomicOr(&kh_lora_index_error, OP_BAD_STARTS);
          ad = -1;
        }
        if (ad >= 0 && fresh && lane == __ffs(peers) - 1) {
          pieces.id[at] = ad;
          pieces.off[at] = make_uint4(~0u, ~0u, ~0u, ~0u);
        }
        __syncwarp();
        if (ad >= 0) {
          uint32_t* off = reinterpret_cast<uint32_t*>(&pieces.off[at]);
#pragma unroll
          for (int w = 0; w < 4; ++w) atomicAnd(off + w, ~lanes_on(lo[j], hi[j], w));
        }
        n = min(n + __popc(added), LISTED);
        __syncwarp();
      }
      more = __all_sync(0xffffffffu, lo[3] < 128);
    }
    const int np = n;
    if (lane == 0) pieces.count = np;
    __syncwarp();
    mbar_arrive(listed);
    const bool lead = elect_one();
    bool ok = true;
    int as = 0;
    uint32_t v = 0, pend = 0;  // pend: two bits a stage: issued, parity
    for (int kb = 0; kb < nk && ok; ++kb)
      for (int i = 0; i < np; ++i) {
        if (!wwait(&a_empty[as], v ^ 1, 202)) { ok = false; break; }
        mbar_arrive_expect_tx_if(lead, &a_full[as], a_bytes);
        tma_load_2d_if(lead, sA + as * a_bytes, &tma, &a_full[as], (kb0 + kb) * 64, pieces.id[i] * p.rank);
        __syncwarp();
        pend = (pend & ~(3u << (2 * as))) | ((2u | v) << (2 * as));
        if (++as == astages) {
          as = 0;
          v ^= 1;
        }
      }
    if (!ok) {
      abort_flag = 1;
      for (int i = 0; i < astages; ++i)
        if ((pend >> (2 * i)) & 2u) mbar_wait(&a_full[i], (pend >> (2 * i)) & 1u, 204);
    }
  } else if (warp == 1) {
    // all lanes in step, one issues
    const uint32_t idesc = idesc_f16(128, R16);
    const bool lead = elect_one();
    bool ok = wwait(listed, 0, 209);
    const int np = ok ? pieces.count : 0;
    int as = 0, xs = 0;
    uint32_t av = 0, xv = 0;
    for (int kb = 0; kb < nk && np && ok; ++kb) {
      if (!wwait(&x_full[xs], xv, 205)) { ok = false; break; }
      const uint64_t dx = desc_sw128(sX + xs * 16384);
      for (int i = 0; i < np; ++i) {
        const uint4 o = pieces.off[i];
        if (!wwait(&a_full[as], av, 206)) { ok = false; break; }
        fence_after_sync();
        const uint64_t da = desc_sw128(sA + as * a_bytes);
        const uint32_t off[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
        for (int k = 0; k < 4; ++k)
          mma_f16_lanes_if(lead, tmem, dx + uint64_t(2 * k), da + uint64_t(2 * k), idesc, (kb | k) ? 1u : 0u, off);
        mma_commit_if(lead, &a_empty[as]);
        __syncwarp();
        if (++as == astages) {
          as = 0;
          av ^= 1;
        }
      }
      mma_commit_if(ok && lead, &x_empty[xs]);
      __syncwarp();
      if (++xs == xstages) {
        xs = 0;
        xv ^= 1;
      }
    }
    if (!ok) {
      abort_flag = 1;
      if (lead) mma_commit(drain);
      __syncwarp();
      mbar_wait(drain, 0, 207);
    }
    if (lead) mma_commit(done);  // (after a failure too: nothing is stored then)
    __syncwarp();
  } else {
    const int quarter = warp & 3, r = quarter * 32 + lane, t = r0 + r;
    bool ok = wwait(listed, 0, 210);
    int ad = -1;
    for (int i = 0, np = ok ? pieces.count : 0; i < np; ++i)
      if (!((reinterpret_cast<const uint32_t*>(&pieces.off[i])[quarter] >> lane) & 1u)) ad = pieces.id[i];
    pieces.row_id[r] = ad;
    const float s = ad >= 0 && p.scales ? __ldg(p.scales + ad) : 1.f;
    pieces.row_scale[r] = s;
    ok = ok && wwait(done, 0, 208) && !abort_flag;
    fence_after_sync();
    if (!ok) ad = -1;
    const bool any = nk > 0 && pieces.count > 0;  // else the accumulator was never written
    const uint32_t taddr = tmem + (uint32_t(quarter * 32) << 16);
    float* part = reinterpret_cast<float*>(smem) + r * (R16 + 4);  // split sums, over the stages (all read)
#pragma unroll 1
    for (int c = 0; c < R16; c += 8) {
      uint32_t v[8];
      tmem_ld8(taddr + uint32_t(c), v);
      tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < 8; ++i) asm volatile("" : "+r"(v[i]));
      if (Z > 1) {
#pragma unroll
        for (int i = 0; i < 8; i += 4)
          *reinterpret_cast<float4*>(part + c + i) =
              any ? make_float4(__uint_as_float(v[i]), __uint_as_float(v[i + 1]), __uint_as_float(v[i + 2]), __uint_as_float(v[i + 3]))
                  : make_float4(0.f, 0.f, 0.f, 0.f);
      } else if (ad >= 0 && c < p.rank) {
        *reinterpret_cast<uint4*>(p.h + int64_t(t) * p.rank + c) =
            make_uint4(pack_half2(__uint_as_float(v[0]) * s, __uint_as_float(v[1]) * s),
                       pack_half2(__uint_as_float(v[2]) * s, __uint_as_float(v[3]) * s),
                       pack_half2(__uint_as_float(v[4]) * s, __uint_as_float(v[5]) * s),
                       pack_half2(__uint_as_float(v[6]) * s, __uint_as_float(v[7]) * s));
      }
    }
  }
  fence_before_sync();
  __syncthreads();
  if (Z > 1) {
    cluster_sync();
    // CTA z adds up rows [z per, (z + 1) per), a thread 4 of a row's values
    const int per = 128 / Z, quads = p.rank / 4;
    const float* base = reinterpret_cast<const float*>(smem);
    for (int e = threadIdx.x; e < per * quads; e += 224) {
      const int r = z * per + e / quads, c = e % quads * 4;
      if (pieces.row_id[r] < 0 || abort_flag) continue;
      const float s = pieces.row_scale[r];
      float4 u[8], v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int q = 0; q < 8; ++q) u[q] = q < Z ? ld_cluster_f32x4(cluster_addr(base + r * (R16 + 4) + c, uint32_t(q))) : v;
#pragma unroll
      for (int q = 0; q < 8; ++q) v.x += u[q].x, v.y += u[q].y, v.z += u[q].z, v.w += u[q].w;
      *reinterpret_cast<uint2*>(p.h + int64_t(r0 + r) * p.rank + c) = make_uint2(pack_half2(v.x * s, v.y * s), pack_half2(v.z * s, v.w * s));
    }
    cluster_sync();
  }
  if (warp == 1) {
    fence_after_sync();
    tmem_free(tmem, cols);
  }
}

// ---- many rows: the projection on CTA pairs ----
//
// 256 x BN tiles of a cluster of two CTAs (tcgen05 cta_group::2: each stages its 128 rows of x and
// BN / 2 rows of W per K block of 64), persistent over the tiles, two accumulators in TMEM so that the
// epilogue runs under the next tile's products. Behind a tile's K blocks come, in the same ring of
// stages, the adapters of its rows: the tile's rows of h against the adapter's rows of B, products of
// ceil(rank / 16) steps whose lanes of other rows are off.
//   warp 0 TMA; warp 1 MMA (first CTA); then a warpgroup per 64 columns: bias, f16, staged and stored by
//   TMA (tiles with rows that are not to be written: straight from registers); the last warp finds the
//   adapters of the tiles ahead, in lists of up to 16 from 32 segments (found by the TMA warp itself, the
//   dependent loads of the search held up the K blocks: 7 % on 65,536 rows of 768 -> 2,304).
// 256 texts of 68,000 rows, 768 -> 2,304, 16 adapters of rank 32: 199 us by itself, 1,270 TFLOP/s, the tensor
// pipe 71 % busy under the power cap; h before it 24 us by itself (its x 4 TB/s). The call: 232 to 270 in a graph.

constexpr int BM = 128;
constexpr int BK = 64;
constexpr int A_BYTES = BM * BK * 2;
constexpr int OUT_BYTES = 128 * 64 * 2;

template <int BN>
struct PCfg {
  static constexpr int BH = BN / 2;
  static constexpr int B_BYTES = BH * BK * 2;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int NWG = BN / 64;
  static constexpr int THREADS = 64 + 128 * NWG + 32;
  static constexpr int STAGES = BN == 256 ? 5 : 6;
  static constexpr uint32_t TMEM_COLS = BN == 128 ? 256 : 512;
  static constexpr int SMEM = STAGES * STAGE_BYTES + NWG * OUT_BYTES + 1024 + 512 + 1280;
};

// What a stage holds for the MMA warp: the lanes an adapter's product leaves alone, its steps of 16,
// whether the tile ends.
struct StageNote {
  uint4 off[2];
  int steps, last, pad[2];
};

// Adapters of a tile and the lanes of other rows; more: the tile has another list.
struct RunList {
  int count, more, pad[2];
  int id[16];
  uint32_t off[16][8];
};

template <int BN>
__global__ void __launch_bounds__(PCfg<BN>::THREADS, 1)
    lora_pair_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW,
                     const __grid_constant__ CUtensorMap tmH, const __grid_constant__ CUtensorMap tmB,
                     const __grid_constant__ CUtensorMap tmO, const LoraParams p) {
  using G = PCfg<BN>;
  constexpr int STAGES = G::STAGES;
  constexpr int NWG = G::NWG;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + STAGES * A_BYTES;
  uint8_t* sOut = sB + STAGES * G::B_BYTES;  // [warpgroup] 16 KB staging tiles
  uint64_t* full = reinterpret_cast<uint64_t*>(sOut + NWG * OUT_BYTES);
  uint64_t* empty = full + STAGES;
  uint64_t* tfull = empty + STAGES;
  uint64_t* tempty = tfull + 2;
  uint64_t* drain = tempty + 2;
  uint64_t* list_full = drain + 2;  // [2]
  uint64_t* list_empty = list_full + 2;
  StageNote* notes = reinterpret_cast<StageNote*>(list_empty + 2);  // [STAGES], 16-byte aligned
  RunList* lists = reinterpret_cast<RunList*>(notes + STAGES);      // [2]
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(lists + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const bool first = rank == 0;
  const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;
  const int begin = seg_start(p, 0), end = seg_start(p, p.n_segs);  // rows to write
  const int m_first = begin / (2 * BM), m_tiles = end > begin ? (end + 2 * BM - 1) / (2 * BM) - m_first : 0;
  const int n_tiles = (p.n + BN - 1) / BN;
  const int tiles = m_tiles * n_tiles;
  const int nk = (p.k + BK - 1) / BK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], 2 * 4 * NWG);  // one arrival per epilogue warp of both CTAs
    }
    mbar_init(drain, 1);
    for (int b = 0; b < 2; ++b) {
      mbar_init(&list_full[b], 1);
      mbar_init(&list_empty[b], 1);
    }
    *abort_flag = 0;
    fence_barrier_init();
    prefetch_tmap(&tmX);
    prefetch_tmap(&tmW);
    prefetch_tmap(&tmO);
  }
  if (warp == 1) tmem_alloc_pair(tmem_holder, G::TMEM_COLS);
  fence_before_sync();
  cluster_sync();  // both CTAs' barriers exist before either signals the other
  fence_after_sync();
  const uint32_t tmem = *tmem_holder;

  if (warp == 0) {
    int stage = 0;
    uint32_t phase = 0;
    uint32_t issued = 0, last_parity = 0;
    bool ok = true, waited = false;
    const bool lead = elect_one();
    const uint32_t full0 = cluster_addr(&full[0], 0);  // both CTAs' bytes complete on the first CTA's barriers
    // One stage, all lanes in step: columns [64 kb, 64 kb + 64) of x and W, or of h and an adapter's
    // rows of B.
    auto emit = [&](const CUtensorMap* ma, const CUtensorMap* mbm, int kb, int row_a, int row_b) {
      mbar_arrive_expect_tx_if(lead && first, &full[stage], 2 * G::STAGE_BYTES);
      const uint32_t bar = full0 + uint32_t(stage) * 8u;
      tma_load_2d_pair_if(lead, sA + stage * A_BYTES, ma, bar, kb * BK, row_a);
      tma_load_2d_pair_if(lead, sB + stage * G::B_BYTES, mbm, bar, kb * BK, row_b);
      issued |= 1u << stage;
      last_parity = (last_parity & ~(1u << stage)) | (phase << stage);
      if (++stage == STAGES) {
        stage = 0;
        phase ^= 1;
      }
    };
    auto room = [&]() -> bool { return __all_sync(0xffffffffu, mbar_wait(&empty[stage], phase ^ 1, 211)); };
    const int chunks = (p.rank + 63) / 64;
    int list = 0;
    uint32_t lphase = 0;
    for (int t = pair; t < tiles && ok; t += npairs) {
      const int mb = m_first + t / n_tiles, nb = t % n_tiles;
      const int row_a = mb * 2 * BM + int(rank) * BM, row_b = nb * BN + int(rank) * G::BH;
      for (int kb = 0; kb + 1 < nk; ++kb) {
        if (!room()) {
          ok = false;
          break;
        }
        emit(&tmX, &tmW, kb, row_a, row_b);
      }
      // A stage is held back until it is known whether another follows it: the MMA warp is told with the
      // last K block and with every run of rows whether the tile ends there.
      int held_kb = nk - 1, held_id = -1;
      uint32_t held_off = 0;  // lane w < 8: word w of the lanes that are off
      auto flush = [&](bool last) {
        if (!ok || !room()) {
          ok = false;
          return;
        }
        if (first) {
          if (held_id >= 0 && lane < 8) reinterpret_cast<uint32_t*>(notes[stage].off)[lane] = held_off;
          if (lane == 8) notes[stage].steps = (min(p.rank - 64 * held_kb, 64) + 15) / 16;
          if (lane == 9) notes[stage].last = last;
          __syncwarp();  // before the arrival that the MMA warp waits for
        }
        if (held_id < 0) emit(&tmX, &tmW, held_kb, row_a, row_b);
        else emit(&tmH, &tmB, held_kb, row_a, held_id * p.n + row_b);
      };
      for (bool more = p.n_adapters > 0; more && ok;) {
        if (!__all_sync(0xffffffffu, mbar_wait(&list_full[list], lphase, 216))) {
          ok = false;
          break;
        }
        const int count = lists[list].count;
        more = lists[list].more != 0;
        if (count > 0 && !waited) {
          wait_primary();  // h is complete
          waited = true;
        }
        for (int i = 0; i < count && ok; ++i) {
          const int id = lists[list].id[i];
          const uint32_t off = lists[list].off[i][lane & 7];
          for (int c = 0; c < chunks && ok; ++c) {
            flush(false);
            held_kb = c;
            held_id = id;
            held_off = off;
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&list_empty[list]);
        if (++list == 2) {
          list = 0;
          lphase ^= 1;
        }
      }
      flush(true);
    }
    if (!ok && lane == 0) {
      *abort_flag = 1;
      // the first CTA's barriers count both CTAs' copies: wait for the ones issued
      if (first)
        for (int s = 0; s < STAGES; ++s)
          if (issued & (1u << s)) mbar_wait(&full[s], (last_parity >> s) & 1u, 221);
    }
    if (!waited) wait_primary();
  } else if (warp == 1) {
    if (first) {  // all lanes in step, one issues
      const uint32_t idesc = idesc_f16(2 * BM, BN);
      const bool lead = elect_one();
      auto wwait = [&](uint64_t* bar, uint32_t parity, int code) -> bool {
        return __all_sync(0xffffffffu, mbar_wait(bar, parity, code));
      };
      const uint64_t da0 = desc_sw128(sA), db0 = desc_sw128(sB);
      int stage = 0;
      uint32_t phase = 0;
      int local = 0;
      bool ok = true;
      for (int t = pair; t < tiles && ok; t += npairs, ++local) {
        const int buf = local & 1;
        const uint32_t tphase = (local >> 1) & 1;
        if (!wwait(&tempty[buf], tphase ^ 1, 212)) {
          ok = false;
          break;
        }
        fence_after_sync();
        const uint32_t d = tmem + uint32_t(buf * BN);
        for (int i = 0;; ++i) {
          if (!wwait(&full[stage], phase, 213)) {
            ok = false;
            break;
          }
          fence_after_sync();
          const uint64_t da = da0 + uint64_t(stage * (A_BYTES >> 4)), db = db0 + uint64_t(stage * (G::B_BYTES >> 4));
          const bool last = i + 1 >= nk && notes[stage].last;
          if (i < nk) {
#pragma unroll
            for (int k = 0; k < BK / 16; ++k)
              mma_f16_pair_if(lead, d, da + uint64_t(k * 2), db + uint64_t(k * 2), idesc, (i | k) != 0 ? 1u : 0u);
            mma_commit_pair_both_if(lead, &empty[stage]);  // the stage is free again in both CTAs
          } else {
            const uint4 o0 = notes[stage].off[0], o1 = notes[stage].off[1];
            const int steps = notes[stage].steps;
            const uint32_t off[8] = {o0.x, o0.y, o0.z, o0.w, o1.x, o1.y, o1.z, o1.w};
#pragma unroll
            for (int k = 0; k < BK / 16; ++k)
              mma_f16_pair_lanes_if(lead && k < steps, d, da + uint64_t(k * 2), db + uint64_t(k * 2), idesc, 1u, off);
            mma_commit_pair_both_if(lead, &empty[stage]);
          }
          __syncwarp();
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1;
          }
          if (last) break;
        }
        if (!ok) break;
        if (lead) mma_commit_pair_both(&tfull[buf]);
        __syncwarp();
      }
      if (!ok) {
        *abort_flag = 1;
        if (lead) mma_commit_pair(drain);  // the MMAs in flight finish before the TMEM is freed
        __syncwarp();
        mbar_wait(drain, 0, 222);
      }
    }
  } else if (warp == 2 + 4 * NWG) {
    if (p.n_adapters > 0) {
      int list = 0;
      uint32_t lphase = 0;
      bool ok = true;
      for (int t = pair; t < tiles && ok; t += npairs) {
        const int r0 = (m_first + t / n_tiles) * 2 * BM, r1 = min(r0 + 2 * BM, end);
        int s = first_seg(p, r0, 32);
        for (bool more = true; more && ok; s += 32) {
          const int i = s + lane;
          int lo = 0, hi = 0, id = -1;
          bool in = i < p.n_segs;
          if (in) {
            lo = max(seg_start(p, i), r0) - r0;
            hi = min(seg_start(p, i + 1), r1) - r0;
            in = r0 + lo < r1;
            if (lo < hi) id = adapter_of(p, i);
          }
          more = __all_sync(0xffffffffu, in);
          // the adapters of these segments, each with all its rows, numbered by their first lanes
          const uint32_t peers = __match_any_sync(0xffffffffu, id);
          const uint32_t firsts = __ballot_sync(0xffffffffu, id >= 0 && lane == __ffs(peers) - 1);
          const int at = __popc(firsts & ((1u << (__ffs(peers) - 1)) - 1u)), count = __popc(firsts);
          if (count == 0 && more) continue;
          for (int base = 0; ok && (base == 0 || base < count); base += 16) {
            ok = __all_sync(0xffffffffu, mbar_wait(&list_empty[list], lphase ^ 1, 215));
            if (!ok) break;
            for (int w = lane; w < 128; w += 32) (&lists[list].off[0][0])[w] = ~0u;
            __syncwarp();
            if (id >= 0 && at >= base && at < base + 16) {
              lists[list].id[at - base] = id;  // (the same from all its lanes)
#pragma unroll
              for (int w = 0; w < 8; ++w) atomicAnd(&lists[list].off[at - base][w], ~lanes_on(lo, hi, w));
            }
            if (lane == 0) {
              lists[list].count = min(count - base, 16);
              lists[list].more = more || base + 16 < count;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&list_full[list]);
            if (++list == 2) {
              list = 0;
              lphase ^= 1;
            }
          }
        }
      }
      if (!ok) *abort_flag = 1;
    } else {  // every id is one that does not exist; no product needs a list
      for (int i = int(blockIdx.x) * 32 + lane; i < p.n_segs; i += int(gridDim.x) * 32)
        if (seg_start(p, i) < seg_start(p, i + 1)) adapter_of(p, i);
    }
  } else {
    const int q = warp & 3;
    const int g = (warp - 2) >> 2;
    const int r = q * 32 + lane;
    const bool leader = (warp == 2 + 4 * g) && lane == 0;
    uint8_t* stile = sOut + g * OUT_BYTES;
    int local = 0;
    for (int t = pair; t < tiles; t += npairs, ++local) {
      const int buf = local & 1;
      const uint32_t tphase = (local >> 1) & 1;
      const int mb = m_first + t / n_tiles, nb = t % n_tiles;
      const int row0 = mb * 2 * BM + int(rank) * BM;  // first row of this CTA's half of the tile
      const int nc = nb * BN + g * 64;
      const bool inside = row0 >= begin && row0 + BM <= end;  // every row is to be written
      if (leader) bulk_wait_read<0>();
      const bool failed = *abort_flag || !mbar_wait(&tfull[buf], tphase, 214);
      if (named_bar_any(1 + g, 128, failed)) {  // (and the staging tile is free)
        *abort_flag = 1;
        break;
      }
      fence_after_sync();
      const uint32_t taddr = tmem + (uint32_t(q * 32) << 16) + uint32_t(buf * BN + g * 64);
      const int row = row0 + r;
      float2 zero = make_float2(0.f, 0.f);  // NaN once an output is infinite or NaN
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t a[32];
        tmem_ld32(taddr + 32 * half, a);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 32; ++i) asm volatile("" : "+r"(a[i]));
        if (half == 1) {  // tells the MMA thread that this warp has read its accumulator rows
          fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(cluster_addr(&tempty[buf], 0));
        }
#pragma unroll
        for (int c8 = 0; c8 < 4; ++c8) {
          const int n = nc + 32 * half + 8 * c8;
          uint4 bias = make_uint4(0, 0, 0, 0);
          if (p.bias && n < p.n) bias = __ldg(reinterpret_cast<const uint4*>(p.bias + n));
          const __half2* bh = reinterpret_cast<const __half2*>(&bias);
          uint32_t u[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 v = fadd2(make_float2(__uint_as_float(a[8 * c8 + 2 * e]), __uint_as_float(a[8 * c8 + 2 * e + 1])),
                                   __half22float2(bh[e]));
            u[e] = pack_half2(v.x, v.y);
            zero = ffma2(v, make_float2(0.f, 0.f), zero);
          }
          const uint4 o = make_uint4(u[0], u[1], u[2], u[3]);
          if (inside) *reinterpret_cast<uint4*>(stile + r * 128 + (((4 * half + c8) ^ (r & 7)) * 16)) = o;
          else if (row >= begin && row < end && n < p.n)
            *reinterpret_cast<uint4*>(p.out + row * p.out_stride + n) = o;
        }
      }
      if (p.n_adapters > 0) {
        uint32_t rows = __ballot_sync(0xffffffffu, zero.x + zero.y != 0.f && row >= begin && row < end);
        __syncwarp();  // (such a row is written again, over what its own lane wrote)
        for (; rows; rows &= rows - 1) {
          const int rr = q * 32 + __ffs(rows) - 1, again = row0 + rr, seg = first_seg(p, again, 0);
          const int ad = seg < p.n_segs && again >= seg_start(p, seg) ? adapter_of(p, seg) : -1;
          if (ad < 0) continue;
          row_beyond_f16(p, again, ad, nc, min(64, p.n - nc), [&](int j, float v) {
            if (lane) return;
            if (inside) *reinterpret_cast<__half*>(stile + rr * 128 + (((j >> 3) ^ (rr & 7)) * 16) + (j & 7) * 2) = __float2half_rn(v);
            else p.out[again * p.out_stride + nc + j] = __float2half_rn(v);
          });
        }
        __syncwarp();
      }
      fence_proxy_async_smem();
      named_bar(1 + g, 128);
      if (leader && inside) {
        if (nc < p.n) tma_store_2d(&tmO, stile, nc, row0);
        bulk_commit();
      }
    }
    if (leader) bulk_wait<0>();
  }
  fence_before_sync();
  cluster_sync();  // neither CTA leaves while the other may still use its shared memory or TMEM
  if (warp == 1) {
    fence_after_sync();
    tmem_free_pair(tmem, G::TMEM_COLS);
  }
}

// ---- host side ----

// CTAs in clusters, one an SM, that surely run at once: the SMs come in groups of 16 to 18, of which a
// cluster of 8 leaves up to two idle (18 clusters of 8 took two rounds: 11 us against 5.8 for 18 of 4, 32
// rows 512 -> 2,304).
constexpr int CLUSTER_CTAS = 128;
constexpr int SMS = 148;

template <class F, class... A>
void launch_ex(F* kernel, dim3 grid, int threads, size_t smem, int cluster, bool dependent, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = unsigned(cluster);
    attr[n].val.clusterDim.y = 1;
    attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (dependent) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.gridDim = grid;
  cfg.blockDim = dim3(unsigned(threads), 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = unsigned(n);
  KH_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...));
}

// Adapters that a tile of 128 rows holds, about: no more than there are, nor than its segments.
int64_t tile_adapters(const kh_lora_matmul_args& a) {
  return std::min<int64_t>({int64_t(a.n_adapters), 128, std::max<int64_t>(1, 128 * int64_t(a.n_segs) / a.rows)});
}
// h by a CTA per row, which reads its adapter's A through L2, instead of by tiles, which take a product
// for each adapter. Few rows (120 of rank 64, 4,096 values to a sum, are too many already: 32 us against
// 28); a few hundred of some adapters (268 rows of 5, 384 -> 768, rank 24: the whole call 16 us against 19;
// 689 of 5, 4,096 -> 384, rank 16, are too many: 32 against 26); some thousand of many (2,000 of 25 to a tile,
// 768 -> 768, rank 16: 39 against 42; 6,000: 69 against 49); any number where a tile would take more products
// than the rank is worth (20,000 single rows, 4,096 -> 4,096, rank 64: 3,154 against 3,537; 64 to a tile, rank 16:
// 1,432 against 1,847, rank 64: 2,561 against 2,045).
bool shrinks_rows(const kh_lora_matmul_args& a) {
  const int64_t work = a.rows * a.rank * int64_t(a.k), adapters = tile_adapters(a);
  return (a.rows <= FT && work <= (1 << 24)) || (adapters > 4 && work <= (1 << 23)) || (adapters >= 16 && work <= (1 << 25)) ||
         (adapters >= 56 && 2 * adapters >= 3 * a.rank);
}
// Rows of x as the columns of the product: W is read once per 128 rows, where a pair's tile takes a product
// for each of its adapters. Up to 128 rows; of many adapters up to four times that (187 rows of 16 adapters,
// 768 -> 384: 18 us against 50; 477 of 23 to a tile 19 against 27, of 16 41 against 27).
bool takes_few(const kh_lora_matmul_args& a) {
  const int64_t blocks = (a.rows + FT - 1) / FT;
  return blocks <= 1 || (blocks <= 4 && tile_adapters(a) >= 5 * blocks);
}
// h from the same launch: every cluster makes it for itself, so A is read once per 128 outputs.
bool fuses(const kh_lora_matmul_args& a) { return takes_few(a) && a.n_adapters > 0 && a.n_adapters * a.rank <= 128; }

template <bool FUSED>
void launch_few(const LoraParams& p, const kh_lora_matmul_args& a, cudaStream_t st) {
  static std::atomic<uint64_t> configured{0};
  once_per_device(configured, [] {
    KH_CUDA(cudaFuncSetAttribute(lora_few_kernel<FUSED>, cudaFuncAttributeMaxDynamicSharedMemorySize, FSMEM + 1024));
  });
  const int cols = int(std::min<int64_t>(FT, (a.rows + 15) / 16 * 16));
  const int stages = std::min(12, FSMEM / ((FUSED ? 32768 : 16384) + cols * 128));
  const int n_tiles = (a.n + 127) / 128, nk = (a.k + 63) / 64;
  // CTAs that split the sum of 128 outputs: while SMs are idle, at least two K blocks each (one: 32 rows
  // 768 -> 768, 9.3 us against 8.8)
  int Z = 1;
  while (Z < 8 && 2 * Z * n_tiles <= CLUSTER_CTAS && 4 * Z <= nk) Z *= 2;
  CUtensorMap tx, tw, ta;
  encode_tensor_map_f16(&tx, a.x, uint64_t(a.rows), uint64_t(a.k), uint64_t(a.x_stride), 64, uint32_t(cols), 128);
  encode_tensor_map_f16(&tw, a.w, uint64_t(a.n), uint64_t(a.k), uint64_t(a.k), 64, 128, 128);
  ta = tw;
  const int a_rows = a.n_adapters * a.rank;
  if (FUSED) encode_tensor_map_f16(&ta, a.lora_a, uint64_t(a_rows), uint64_t(a.k), uint64_t(a.k), 64, uint32_t(a_rows), 128);
  const dim3 grid(unsigned(n_tiles * Z), unsigned((a.rows + FT - 1) / FT));
  launch_ex(lora_few_kernel<FUSED>, grid, FTHREADS, FSMEM + 1024, Z, !FUSED && a.n_adapters > 0, st, tx, tw, ta, p, Z, cols,
            stages, a_rows * 128);
}

template <int BN>
void launch_pair(const LoraParams& p, const kh_lora_matmul_args& a, bool dependent, cudaStream_t st) {
  using G = PCfg<BN>;
  static std::atomic<uint64_t> configured{0};
  once_per_device(configured, [] {
    KH_CUDA(cudaFuncSetAttribute(lora_pair_kernel<BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, G::SMEM));
  });
  CUtensorMap tx, tw, th, tb, to;
  encode_tensor_map_f16(&tx, a.x, uint64_t(a.rows), uint64_t(a.k), uint64_t(a.x_stride), BK, BM, 128);
  encode_tensor_map_f16(&tw, a.w, uint64_t(a.n), uint64_t(a.k), uint64_t(a.k), BK, G::BH, 128);
  encode_tensor_map_f16(&to, a.out, uint64_t(a.rows), uint64_t(a.n), uint64_t(a.out_stride), 64, BM, 128);
  th = tb = tw;  // (without adapters neither is read)
  if (a.n_adapters) {
    encode_tensor_map_f16(&th, a.workspace, uint64_t(a.rows), uint64_t(a.rank), uint64_t(a.rank), BK, BM, 128);
    encode_tensor_map_f16(&tb, a.lora_b, uint64_t(a.n_adapters) * a.n, uint64_t(a.rank), uint64_t(a.rank), BK, G::BH, 128);
  }
  const int64_t tiles = (a.rows + 2 * BM - 1) / (2 * BM) * ((a.n + BN - 1) / BN);
  const int pairs = int(std::min<int64_t>(tiles, device_sms() / 2));
  launch_ex(lora_pair_kernel<BN>, dim3(unsigned(2 * pairs)), G::THREADS, G::SMEM, 2, dependent, st, tx, tw, th, tb, to, p);
}

void check_sizes(const char* fn, const kh_lora_matmul_args* args) {
  check_that(args != nullptr, fn, "null arguments");
  const kh_lora_matmul_args& a = *args;
  check_that(a.k >= 8 && a.k <= 65536 && a.k % 8 == 0 && a.n >= 8 && a.n <= 65536 && a.n % 8 == 0, fn,
             "k and n must be multiples of 8, in [8, 65536]");
  check_that(a.rank >= 8 && a.rank <= 128 && a.rank % 8 == 0, fn, "rank must be a multiple of 8, in [8, 128]");
  check_that(a.n_adapters >= 0 && a.n_adapters <= 65535 && int64_t(a.n_adapters) * a.n < (int64_t(1) << 31) - 512, fn,
             "n_adapters must be in [0, 65535], n_adapters * n below 2^31 - 512");
  check_that(a.n_segs >= 0 && a.n_segs <= 65535, fn, "n_segs must be in [0, 65535]");
  check_that(a.rows >= 0 && a.rows < (int64_t(1) << 31) - 256, fn, "rows must be in [0, 2^31 - 256)");
}

}  // namespace

int64_t lora_matmul_workspace(const kh_lora_matmul_args* args) {
  check_sizes("kh_lora_matmul_f16_workspace", args);
  // (the same whichever kernels take the call, so that a workspace for the most rows serves fewer)
  return args->n_adapters ? args->rows * args->rank * 2 : 0;
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
  check_that(aligned4(a.scales) && aligned4(a.seg_starts) && aligned4(a.seg_adapters), fn,
             "scales, seg_starts and seg_adapters must be 4-byte aligned");
  const int64_t lim = int64_t(1) << 31;
  check_that(a.x_stride >= a.k && a.out_stride >= a.n && a.x_stride < lim && a.out_stride < lim &&
                 a.x_stride % 8 == 0 && a.out_stride % 8 == 0,
             fn, "strides must be multiples of 8, at least k and n, below 2^31");
  check_that(a.x != a.out, fn, "out may not be x: every row of x is read for all outputs");
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
  const bool adapters = a.n_adapters > 0;
  if (adapters && !fuses(a)) {
    if (shrinks_rows(a)) {
      // (with the next kernel's split of an SM's memory, so that its CTAs may start beside these)
      static std::atomic<uint64_t> configured{0};
      once_per_device(configured, [] {
        KH_CUDA(cudaFuncSetAttribute(lora_shrink_rows_kernel, cudaFuncAttributePreferredSharedMemoryCarveout,
                                     cudaSharedmemCarveoutMaxShared));
      });
      lora_shrink_rows_kernel<<<unsigned(a.rows), 512, 0, st>>>(p);
      KH_CUDA(cudaGetLastError());
    } else {
      const int R16 = (a.rank + 15) / 16 * 16;
      static std::atomic<uint64_t> configured{0};
      once_per_device(configured, [] {
        KH_CUDA(cudaFuncSetAttribute(lora_shrink_tile_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     SXS * 16384 + 4 * 128 * 128 + 1024));
      });
      CUtensorMap tx, ta;
      encode_tensor_map_f16(&tx, a.x, uint64_t(a.rows), uint64_t(a.k), uint64_t(a.x_stride), 64, 128, 128);
      encode_tensor_map_f16(&ta, a.lora_a, uint64_t(a.n_adapters) * a.rank, uint64_t(a.k), uint64_t(a.k), 64, R16, 128);
      const int64_t tiles = (a.rows + 127) / 128;
      int Z = 1;  // CTAs that split a tile's sum: while SMs are idle, at least two K blocks each
      // (two CTAs an SM up to rank 32: 43 tiles of 1,536 -> 384, rank 16, the whole call 22 us against 24 with
      // a bound of 128 CTAs and 26 with 400)
      const int at_once = R16 <= 32 ? 2 * CLUSTER_CTAS : CLUSTER_CTAS;
      while (Z < 8 && 2 * Z * tiles <= at_once && 4 * Z <= (a.k + 63) / 64) Z *= 2;
      // many tiles: rings so short that four CTAs share an SM (up to rank 32) and cover each other's waits
      const int xstages = tiles > 2 * SMS ? 2 : SXS, astages = R16 > 32 || tiles > 2 * SMS ? 4 : SAS;
      const size_t smem = size_t(xstages) * 16384 + size_t(astages) * R16 * 128 + 1024;
      // Clusters that share a tile's adapters (120 rows of 4 adapters of rank 64, 4,096 -> 4,096, the whole call
      // 27 us against 34 with one), on SMs that the next kernel does not need: 689 rows of 5, 4,096 -> 384,
      // rank 16, 26 us, on all SMs 32.
      const int64_t next = takes_few(a) ? 8 * ((a.n + 127) / 128) : 2 * ((a.rows + 255) / 256) * ((a.n + 191) / 192);
      const int64_t room = next >= CLUSTER_CTAS ? at_once : std::min<int64_t>(at_once, SMS - next);
      int groups = 1;
      while (groups < 8 && 2 * groups * Z * tiles <= room && 2 * groups <= tile_adapters(a)) groups *= 2;
      launch_ex(lora_shrink_tile_kernel, dim3(unsigned(Z * tiles), unsigned(groups)), 224, smem, Z, false, st, tx, ta, p, Z, groups,
                xstages, astages);
    }
  }
  if (takes_few(a)) {
    if (fuses(a)) launch_few<true>(p, a, st);
    else launch_few<false>(p, a, st);
  } else {
    // The tile width that is over soonest: a tile costs its columns and, as a constant, what it reads of x and
    // its adapters' products; a last round that is not full counts in part, as pairs start one after another
    // and the first ones have the tile more (24 texts of 4,254 rows, 768 -> 2,304, 2.07 rounds of 256 columns
    // or 2.76 of 192: 25.5 us against 28.5; 9,974 rows 1,024 -> 1,152: 128 columns 40.6, 192 35.6, 256 36.5).
    const double m_tiles = double((a.rows + 255) / 256), pairs = device_sms() / 2;
    auto cost = [&](int bn) {
      const double rounds = std::max(1.0, m_tiles * ((a.n + bn - 1) / bn) / pairs);
      return (rounds + (rounds < 2 ? 0.35 : 0.15) * (std::ceil(rounds) - rounds)) * (bn + (adapters ? 80 : 24));
    };
    if (cost(256) <= cost(192) && cost(256) <= cost(128)) launch_pair<256>(p, a, adapters, st);
    else if (cost(192) <= cost(128)) launch_pair<192>(p, a, adapters, st);
    else launch_pair<128>(p, a, adapters, st);
  }
}

int* lora_wait_word() {
  void* p = nullptr;
  KH_CUDA(cudaGetSymbolAddress(&p, sm100::kh_tc_error));
  return static_cast<int*>(p);
}

int* lora_index_word() {
  void* p = nullptr;
  KH_CUDA(cudaGetSymbolAddress(&p, kh_lora_index_error));
  return static_cast<int*>(p);
}

}  // namespace kh
