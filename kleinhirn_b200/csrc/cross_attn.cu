// Cross attention of packed query rows over an encoder's packed states of another length.
//
// For query row i of sequence s and query head h, with G = q_heads / kv_heads and K the kept states of
// s: out = sum_j p_j v_j, p the softmax over j in K of scale q_i,h . k_j,h/G; zero where K is empty.
// Both kernels make one pass over the states with a running reference point m (log2 units) and the sum
// l of p = 2^(s - m + LIFT): m moves only when a score exceeds it by more than RISE, so the accumulated output
// is rescaled seldom. p is f16 as the operand of the product with v: at most 2^(LIFT + RISE + 1), rounded by
// 2^-11, and below 2^-14 by up to 2^-25, which is 2^-32 of the largest (m is a score, so the largest p is
// 2^LIFT or more); l adds the f32 values. m, l, scores and the output accumulate in f32.
// The G query heads of a key head are rows of the same tile (row = query * G + head), so k and v are
// read once for them.
//
// Which kernel: see takes_rows_kernel. Few rows to a key head (single tokens): bound by reading k and v
// once, cross_rows_kernel. More: tensor-core products of 128 rows, cross_tile_kernel. Where the rows
// leave SMs idle, the states of a sequence are split over CTAs, whose partial (m, l, O) the workspace
// holds and cross_join_kernel adds up in a fixed order.

#include "device_ops.h"

#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>

#include "runtime.h"
#include "sm100.cuh"
#include "tmap.h"

namespace kh {

namespace {

using namespace sm100;

constexpr float LIFT = 7.f, RISE = 7.f;  // (m - LIFT may round to m - 8: 2^15 at most)

struct CrossParams {
  const __half* q;
  const __half* k;
  const __half* v;
  __half* out;
  const float* mask;
  const int32_t* q_starts;
  const int32_t* k_starts;
  float* part_o;   // [nsplit][n_seqs * max_q][q_heads][D]
  float2* part_ml; // [nsplit][n_seqs * max_q][q_heads]: m, l
  int64_t q_rows, kv_rows, q_stride, k_stride, v_stride, out_stride;
  int n_seqs, q_heads, kv_heads, G, max_q, max_k, nsplit;
  float scale_log2;  // scale * log2(e)
  bool wide;         // 16 columns of out are aligned to their 32 bytes
};

// Rows of sequence s in a buffer of `rows`: starts outside it are cut, a longer sequence ends at `most`.
__device__ __forceinline__ void seq_range(const int32_t* starts, int s, int64_t rows, int most, int64_t& r0, int& n) {
  r0 = min(max(int64_t(starts[s]), int64_t(0)), rows);
  const int64_t r1 = min(max(int64_t(starts[s + 1]), r0), rows);
  n = int(min(r1 - r0, int64_t(most)));
}

// Where the partial result of query i of sequence s, head h, split z lies.
__device__ __forceinline__ int64_t part_index(const CrossParams& p, int z, int s, int i, int h) {
  return ((int64_t(z) * p.n_seqs + s) * p.max_q + i) * p.q_heads + h;
}

// ---- few rows: one m16 block on mma.sync ----
//
// One CTA of RW warps per (split, key head, sequence), rows <= 16 as one m16 block. Each warp has a ring
// of its own, filled by TMA with boxes of 16 states of K and V, and no other warp to wait for until the
// end. A step of 16 states: S = Q K^T in m16n8k16 products, then O += P V with S's accumulator layout as
// P's operand layout. The sum over the head's values and the order of the output columns are free, so a
// thread takes 16-byte pieces of k and v as they lie: within 32 values of k, the quad lane t holds values
// 8 t .. 8 t + 7 of q and k alike; of v, it holds the D / 8 values (lane / 4) D / 8 .. of its four states.
// Bound: HBM (2 D 2 bytes per state and key head, each read once), by the bytes in flight: 64 requests of
// one query on 200-512 states, 12 heads of 64, took 25 us with loads one step ahead in registers.

constexpr int RSTEP = 16;  // states of a step

template <int D, int RW>
struct RCfg {
  static constexpr int STAGES = D == 128 ? 3 : 4;
  static constexpr int PANELS = D == 128 ? 2 : 1, PCOLS = D / PANELS, ROWB = PCOLS * 2;
  static constexpr int PANEL = RSTEP * ROWB, TILE = PANELS * PANEL;  // 16 rows of k or v
  static constexpr int RING = STAGES * 2 * TILE;                     // of a warp
  static constexpr int PART = RW * 16 * (D + 4) * 4;                 // the warps' O at the end, over the rings
  static constexpr int SMEM = (RW * RING > PART ? RW * RING : PART) + 1024;
  // byte offset of 16-byte piece c of row r in a swizzled tile
  static __device__ __forceinline__ int at(int r, int c) {
    if (D == 32) return r * 64 + ((c ^ ((r >> 1) & 3)) * 16);
    return (c >> 3) * PANEL + r * 128 + (((c & 7) ^ (r & 7)) * 16);
  }
};

template <int D, int RW>
__global__ void __launch_bounds__(RW * 32)
    cross_rows_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv, const CrossParams p) {
  using C = RCfg<D, RW>;
  constexpr int E = D / 8;  // output columns of 8 at a time
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t bars[RW][C::STAGES];
  __shared__ float sm[RW][16], sl[RW][16];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = blockIdx.x, hk = blockIdx.y, s = blockIdx.z;
  launch_dependents();
  if (lane == 0) {
    for (int i = 0; i < C::STAGES; ++i) mbar_init(&bars[warp][i], 1);
    fence_barrier_init();
    if (warp == 0) {
      prefetch_tmap(&tmk);
      prefetch_tmap(&tmv);
    }
  }
  __syncwarp();
  int64_t q0, k0;
  int nq, nk;
  seq_range(p.q_starts, s, p.q_rows, p.max_q, q0, nq);
  seq_range(p.k_starts, s, p.kv_rows, p.max_k, k0, nk);
  const int rows = nq * p.G;  // <= 16
  if (rows == 0) return;
  // states of this split, in whole steps
  const int per = ((nk + p.nsplit - 1) / p.nsplit + RSTEP - 1) / RSTEP * RSTEP;
  const int begin = min(split * per, nk), end = min(begin + per, nk);
  const int steps = ((end - begin + RSTEP - 1) / RSTEP - warp + RW - 1) / RW;  // of this warp: warp, warp + RW, ..

  uint8_t* ring = smem + warp * C::RING;
  auto load = [&](int i) {  // step i of this warp into its stage
    if (lane == 0) {
      const int st = i % C::STAGES, y = int(k0) + begin + (i * RW + warp) * RSTEP;
      uint64_t* bar = &bars[warp][st];
      mbar_arrive_expect_tx(bar, 2 * C::TILE);
      for (int c = 0; c < C::PANELS; ++c) {
        tma_load_2d(ring + st * 2 * C::TILE + c * C::PANEL, &tmk, bar, hk * D + c * C::PCOLS, y);
        tma_load_2d(ring + st * 2 * C::TILE + C::TILE + c * C::PANEL, &tmv, bar, hk * D + c * C::PCOLS, y);
      }
    }
  };
  for (int i = 0; i < min(steps, C::STAGES); ++i) load(i);

  // A operand: rows lane / 4 and lane / 4 + 8
  uint32_t qa[D / 32][2][4];
#pragma unroll
  for (int c = 0; c < D / 32; ++c)
#pragma unroll
    for (int hl = 0; hl < 2; ++hl) {
      const int r = (lane >> 2) + 8 * hl;
      uint4 u = make_uint4(0, 0, 0, 0);
      if (r < rows)
        u = *reinterpret_cast<const uint4*>(p.q + (q0 + r / p.G) * p.q_stride + (hk * p.G + r % p.G) * D + c * 32 +
                                            (lane & 3) * 8);
      qa[c][hl][0] = u.x;
      qa[c][hl][1] = u.y;
      qa[c][hl][2] = u.z;
      qa[c][hl][3] = u.w;
    }

  const float* mb = p.mask ? p.mask + k0 : nullptr;
  float o[E][4];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e][0] = o[e][1] = o[e][2] = o[e][3] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};  // rows lane / 4 and + 8; l of this thread's states
  bool ok = true;
  int used = 0;  // steps whose loads have been waited for
  for (int i = 0; i < steps; ++i) {
    const int st = i % C::STAGES, first = begin + (i * RW + warp) * RSTEP;
    bool keep[2][2];
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int j = first + 8 * b + (lane & 3) * 2 + e;
        keep[b][e] = j < end && (!mb || __ldg(mb + j) > 0.5f);
      }
    if (!__all_sync(0xffffffffu, mbar_wait(&bars[warp][st], uint32_t(i / C::STAGES) & 1, 120))) {
      ok = false;
      break;
    }
    ++used;
    const uint8_t* tk = ring + st * 2 * C::TILE;
    const uint8_t* tv = tk + C::TILE;
    float sc[2][4];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      sc[b][0] = sc[b][1] = sc[b][2] = sc[b][3] = 0.f;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        const uint4 kk = *reinterpret_cast<const uint4*>(tk + C::at(8 * b + (lane >> 2), 4 * c + (lane & 3)));
        mma_16816(sc[b], qa[c][0][0], qa[c][1][0], qa[c][0][1], qa[c][1][1], kk.x, kk.y);
        mma_16816(sc[b], qa[c][0][2], qa[c][1][2], qa[c][0][3], qa[c][1][3], kk.z, kk.w);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) sc[b][e] = keep[b][e & 1] ? sc[b][e] * p.scale_log2 : -INFINITY;
    }
    // v of this thread's states; a dropped one's values stay out of the sums whatever they hold
    uint32_t v[2][2][D / 16];
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = 8 * b + (lane & 3) * 2 + e;
        if constexpr (D == 32) {
          const uint2 u = *reinterpret_cast<const uint2*>(tv + C::at(r, lane >> 3) + ((lane >> 2) & 1) * 8);
          v[b][e][0] = keep[b][e] ? u.x : 0u;
          v[b][e][1] = keep[b][e] ? u.y : 0u;
        } else {
#pragma unroll
          for (int c = 0; c < D / 64; ++c) {
            const uint4 u = *reinterpret_cast<const uint4*>(tv + C::at(r, (lane >> 2) * (D / 64) + c));
            v[b][e][4 * c] = keep[b][e] ? u.x : 0u;
            v[b][e][4 * c + 1] = keep[b][e] ? u.y : 0u;
            v[b][e][4 * c + 2] = keep[b][e] ? u.z : 0u;
            v[b][e][4 * c + 3] = keep[b][e] ? u.w : 0u;
          }
        }
      }
    __syncwarp();  // the stage has been read
    if (i + C::STAGES < steps) load(i + C::STAGES);
    float top[2];
#pragma unroll
    for (int r = 0; r < 2; ++r)
      top[r] = fmaxf(fmaxf(sc[0][2 * r], sc[0][2 * r + 1]), fmaxf(sc[1][2 * r], sc[1][2 * r + 1]));
    if (__any_sync(0xffffffffu, top[0] - m[0] > RISE || top[1] - m[1] > RISE)) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
        top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
        const bool moves = top[r] - m[r] > RISE;  // the row's own: another one's scores leave its bits alone
        const float corr = moves ? ex2_approx(m[r] - top[r]) : 1.f;  // (0 from m = -inf)
        if (moves) m[r] = top[r];
        l[r] *= corr;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          o[e][2 * r] *= corr;
          o[e][2 * r + 1] *= corr;
        }
      }
    }
    const float ref[2] = {m[0] == -INFINITY ? 0.f : m[0] - LIFT, m[1] == -INFINITY ? 0.f : m[1] - LIFT};
    uint32_t pa[2][2];
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float x0 = ex2_approx(sc[b][2 * r] - ref[r]), x1 = ex2_approx(sc[b][2 * r + 1] - ref[r]);
        l[r] += x0 + x1;
        pa[b][r] = pack_half2(x0, x1);
      }
#pragma unroll
    for (int e2 = 0; e2 < E / 2; ++e2) {
      // columns 2 e2 and 2 e2 + 1 of the thread's v values: pairs of states side by side
      const uint32_t u0 = v[0][0][e2], u1 = v[0][1][e2], w0 = v[1][0][e2], w1 = v[1][1][e2];
      mma_16816(o[2 * e2], pa[0][0], pa[0][1], pa[1][0], pa[1][1], __byte_perm(u0, u1, 0x5410), __byte_perm(w0, w1, 0x5410));
      mma_16816(o[2 * e2 + 1], pa[0][0], pa[0][1], pa[1][0], pa[1][1], __byte_perm(u0, u1, 0x7632),
                __byte_perm(w0, w1, 0x7632));
    }
  }
  if (!ok)  // every copy this warp issued lands before the rings are used again
    for (int i = used; i < min(steps, used + C::STAGES); ++i) mbar_wait(&bars[warp][i % C::STAGES], uint32_t(i / C::STAGES) & 1, 121);
  __syncthreads();
  float* so = reinterpret_cast<float*>(smem);  // [warp][16][D + 4]
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    const int row = (lane >> 2) + 8 * r;
    if ((lane & 3) == 0) {
      sm[warp][row] = m[r];
      sl[warp][row] = l[r];
    }
    if (row < rows) {
      // column n = 2 (lane & 3) + i of block e is output value n E + e
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < E; e += 4)
          *reinterpret_cast<float4*>(so + (warp * 16 + row) * (D + 4) + (2 * (lane & 3) + i) * E + e) =
              make_float4(o[e][2 * r + i], o[e + 1][2 * r + i], o[e + 2][2 * r + i], o[e + 3][2 * r + i]);
    }
  }
  __syncthreads();
  // the warps' parts, 8 output values of a row per thread
  for (int t = threadIdx.x; t < rows * (D / 8); t += RW * 32) {
    const int row = t / (D / 8), d = t % (D / 8) * 8;
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < RW; ++w) mm = fmaxf(mm, sm[w][row]);
    float lt = 0.f, acc[8] = {};
#pragma unroll
    for (int w = 0; w < RW; ++w) {
      const float f = sm[w][row] == -INFINITY ? 0.f : ex2_approx(sm[w][row] - mm);
      lt += f * sl[w][row];
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] += f * so[(w * 16 + row) * (D + 4) + d + i];
    }
    const int qi = row / p.G, h = hk * p.G + row % p.G;
    if (p.nsplit == 1) {
      const float inv = lt == 0.f ? 0.f : 1.f / lt;
      uint32_t u[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) u[i] = pack_half2(acc[2 * i] * inv, acc[2 * i + 1] * inv);
      *reinterpret_cast<uint4*>(p.out + (q0 + qi) * p.out_stride + h * D + d) = make_uint4(u[0], u[1], u[2], u[3]);
    } else {
      const int64_t at = part_index(p, split, s, qi, h);
      float4* dst = reinterpret_cast<float4*>(p.part_o + at * D + d);
      dst[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
      dst[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
      if (d == 0) p.part_ml[at] = make_float2(mm, lt);
    }
  }
}

// ---- joining the splits: WARPS warps per (query, head), each every WARPS-th split ----
//
// CTAs of 4 warps, launched while the parts are made. Few rows: 4 warps to one, for the loads in flight. Many:
// one (11 sequences of up to 660 queries, heads of 128, 3 splits: 22.8 us with the parts, 28.9 with 4).

template <int D, int WARPS>
__global__ void __launch_bounds__(128) cross_join_kernel(const CrossParams p, int64_t rows) {
  constexpr int V = D / 32;
  __shared__ float so[4][D], sl[4];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t t = int64_t(blockIdx.x) * (4 / WARPS) + warp / WARPS;
  const int64_t per_seq = int64_t(p.max_q) * p.q_heads;
  const int s = int(t / per_seq);
  const int i = int((t - s * per_seq) / p.q_heads), h = int(t % p.q_heads);
  int64_t q0 = 0;
  int nq = 0;
  if (t < rows) seq_range(p.q_starts, s, p.q_rows, p.max_q, q0, nq);
  wait_primary();
  const bool in = i < nq;  // (WARPS 4: the same for the CTA)
  float o[V] = {}, l = 0.f;
  if (in) {
    // the largest reference point first (a lane per split), then the sums, with independent loads
    float m = -INFINITY;
    for (int z = lane; z < p.nsplit; z += 32) m = fmaxf(m, p.part_ml[part_index(p, z, s, i, h)].x);
    for (int w = 16; w; w >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, w));
#pragma unroll 4
    for (int z = warp % WARPS; z < p.nsplit; z += WARPS) {
      const int64_t at = part_index(p, z, s, i, h);
      const float2 ml = p.part_ml[at];
      float v[V];
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = p.part_o[at * D + lane * V + e];
      const float f = ml.x == -INFINITY ? 0.f : ex2_approx(ml.x - m);
      l += f * ml.y;
#pragma unroll
      for (int e = 0; e < V; ++e) o[e] += f == 0.f ? 0.f : f * v[e];  // (without a kept state O holds anything)
    }
  }
  if (WARPS > 1) {
#pragma unroll
    for (int e = 0; e < V; ++e) so[warp][lane * V + e] = o[e];
    if (lane == 0) sl[warp] = l;
    __syncthreads();
    if (warp > 0) return;
    l = (sl[0] + sl[1]) + (sl[2] + sl[3]);
#pragma unroll
    for (int e = 0; e < V; ++e)
      o[e] = (so[0][lane * V + e] + so[1][lane * V + e]) + (so[2][lane * V + e] + so[3][lane * V + e]);
  }
  if (!in) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  __half* dst = p.out + (q0 + i) * p.out_stride + h * D + lane * V;
  if constexpr (V == 1) {
    dst[0] = __float2half_rn(o[0] * inv);
  } else {
#pragma unroll
    for (int e = 0; e < V; e += 2) reinterpret_cast<uint32_t*>(dst)[e / 2] = pack_half2(o[e] * inv, o[e + 1] * inv);
  }
}

// ---- tiles of 128 rows on the tensor cores ----
//
// One CTA per (block of row tiles, key head and split, sequence):
//   warp 0     TMA: Q once, tiles of KEYS states of K and V into two rings; it also clears the dropped
//              states' rows of V tiles (past the end, masked) before they are used;
//   warp 1     issues S = Q K^T (M 128, N KEYS, K = D) into the stream's TMEM columns and O += P V (A = P
//              from TMEM, V as an MN-major operand) into its O columns;
//   8 warps    softmax, four to a stream, one thread per row: its KEYS scores in registers, P (f16)
//              written over S in TMEM.
// The two streams are two row tiles over the same K and V tiles (see row_tiles); where the CTA's rows fit
// one tile, they take its even and odd key tiles instead and add up their (m, l, O) at the end. S of the next
// tile is issued behind P V of the last one, in order, so P may lie over S, and a full S means that the
// products before it are done; one stream's softmax runs under the other's products.
// Key tiles with dropped states: their scores become -inf and their V rows zero in shared memory, so
// that nothing they hold reaches a sum. (Cleared by the softmax warps, which then wait for V and fence:
// 74 us against 62, 301-499 queries on 700-1,500 states with one in seven masked, 16 sequences.)
//
// Bound: the softmax threads. A row tile of 128 x 128 scores takes the special-function unit 1,024
// cycles (4 lanes a clock on each quarter of the SM), its products 512 (D 64) or 1,024 (D 128). Heads of
// 128 fill TMEM with one CTA per SM (KEYS 128; 168 registers a thread are dealt again, so that a softmax
// thread holds its row); smaller heads run two CTAs per SM (KEYS 64, one row tile each: 16 heads of 64,
// 2,048 queries on 4,096 states, 186 us against 202 with two), whose four softmax warps on each quarter
// cover one another's waits, and one CTA's end the other's beginning. (Some of the exponentials by a
// polynomial on the FMA pipe instead: no faster, as the clock falls with the power they take.)

constexpr int TROWS = 128;
constexpr float EXACT_REF = 4194304.f;  // half a unit of 2^22 in the last place: 2^-2

template <int D>
struct TCfg {
  static constexpr bool ONE = D == 128;              // one CTA per SM
  static constexpr int KEYS = ONE ? 128 : 64;
  static constexpr int HALVES = ONE ? 2 : 1;         // parts in which P goes into its products
  static constexpr int FIRST = ONE ? 4 : 2;          // first softmax warp (setmaxnreg acts on whole warpgroups)
  static constexpr int THREADS = 32 * (FIRST + 8);
  // 56 x 128 + 224 x 256 = 168 x 384, the registers of the launch
  static constexpr int REGS_ISSUE = 56, REGS_SOFTMAX = 224;  // (ONE)
  static constexpr int PANELS = ONE ? 2 : 1;         // columns of a swizzled row: 64 (D 32: 32)
  static constexpr int PCOLS = D / PANELS;
  static constexpr int ROWB = PCOLS * 2;             // bytes of a row of a panel: the swizzle width
  static constexpr int QPANEL = TROWS * ROWB, QTILE = PANELS * QPANEL;
  static constexpr int KPANEL = KEYS * ROWB, KTILE = PANELS * KPANEL;
  static constexpr int KS = ONE ? 3 : 4, VS = ONE ? 2 : 4;  // ring stages
  // (a CTA of one row tile exchanges its streams' m and l in the second one's space)
  static constexpr int K_OFF = 2 * QTILE;
  static constexpr int V_OFF = K_OFF + KS * KTILE;
  static constexpr int BAR_OFF = V_OFF + VS * KTILE;
  static constexpr int USED = BAR_OFF + 320 + 1024;
  // as much as keeps a third CTA (its TMEM) off the SM
  static constexpr int SMEM = ONE || USED > 100 * 1024 ? USED : 100 * 1024;
  static constexpr uint32_t S_STRIDE = ONE ? 128 : 64;      // TMEM: S of the streams, then O
  static constexpr uint32_t O_COL = 2 * S_STRIDE, COLS = ONE ? 512 : 256;
  static constexpr uint64_t LAYOUT = D == 32 ? 4ull : 2ull;  // 64- or 128-byte swizzle
  static constexpr uint64_t SBO = (8 * ROWB) >> 4;
  static constexpr uint64_t LBO = PANELS == 2 ? (KPANEL >> 4) : 1ull;  // MN-major V: from panel to panel
};

template <int D>
__device__ __forceinline__ uint64_t tile_desc(const void* smem) {
  using C = TCfg<D>;
  return ((uint64_t(smem_u32(smem)) >> 4) & 0x3FFFull) | (C::LBO << 16) | (C::SBO << 32) | (1ull << 46) | (C::LAYOUT << 61);
}

// 32 aligned bytes, a whole sector, in one store.
__device__ __forceinline__ void store_32(void* dst, const uint32_t (&u)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]),
               "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7])
               : "memory");
}

__device__ __forceinline__ float2 twice(float a) { return make_float2(a, a); }

// Values that tcgen05.ld wrote may be used from here on (the compiler keeps uses behind this).
template <int N>
__device__ __forceinline__ void settle(uint32_t (&r)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i]));
}

// Barrier of the two warps of a quarter. The ids are constants: with an id in a register a CTA counts as
// using all 16 barriers, and a second one does not fit the SM.
__device__ __forceinline__ bool quarter_any(int quarter, bool pred) {
  switch (quarter) {
    case 0: return named_bar_any<1>(64, pred);
    case 1: return named_bar_any<2>(64, pred);
    case 2: return named_bar_any<3>(64, pred);
    default: return named_bar_any<4>(64, pred);
  }
}

// ROW_TILES: of a CTA, at most.
template <int D, int ROW_TILES>
__global__ void __launch_bounds__(TCfg<D>::THREADS, TCfg<D>::ONE ? 1 : 2)
    cross_tile_kernel(const __grid_constant__ CUtensorMap tmq, const __grid_constant__ CUtensorMap tmk,
                      const __grid_constant__ CUtensorMap tmv, const CrossParams p) {
  using C = TCfg<D>;
  constexpr int KEYS = C::KEYS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sK = smem + C::K_OFF;
  uint8_t* sV = smem + C::V_OFF;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::BAR_OFF);
  uint64_t* q_full = bars;
  uint64_t* s_full = bars + 1;         // [stream]
  uint64_t* p_full = bars + 3;         // [stream][half]
  uint64_t* o_full = bars + 7;         // [stream]
  uint64_t* drain = bars + 9;
  uint64_t* v_tail = bars + 10;        // without a mask: the last tile's rows are cleared
  uint64_t* k_full = bars + 11;        // [KS]
  uint64_t* k_empty = k_full + C::KS;
  uint64_t* v_full = k_empty + C::KS;  // [VS]
  uint64_t* v_empty = v_full + C::VS;
  uint64_t* v_clear = v_empty + C::VS;  // [VS] with a mask: the stage's dropped rows are cleared
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(v_clear + C::VS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);

  launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int hk = blockIdx.y % p.kv_heads, split = blockIdx.y / p.kv_heads, s = blockIdx.z;
  const int G = p.G, qpt = TROWS / G;  // queries of a row tile
  int64_t q0, k0;
  int nq, nk;
  seq_range(p.q_starts, s, p.q_rows, p.max_q, q0, nq);
  seq_range(p.k_starts, s, p.kv_rows, p.max_k, k0, nk);
  const int qb = blockIdx.x * ROW_TILES * qpt;  // first query of the CTA
  if (qb >= nq) return;
  const bool pair = ROW_TILES == 2 && nq - qb > qpt;  // two row tiles (else the streams share one tile's states)
  // key tiles of this split
  const int all = (nk + KEYS - 1) / KEYS, per = (all + p.nsplit - 1) / p.nsplit;
  const int t0 = min(split * per, all), nkt = min(t0 + per, all) - t0;
  const int n0_of = pair ? nkt : (nkt + 1) / 2, n1_of = pair ? nkt : nkt / 2;  // tiles of the streams
  auto load_tile = [&](int j, bool is_v) {  // of K or V into its ring, by one thread
    const int st = is_v ? j % C::VS : j % C::KS;
    uint64_t* full = is_v ? &v_full[st] : &k_full[st];
    mbar_arrive_expect_tx(full, C::KTILE);
    uint8_t* dst = (is_v ? sV : sK) + st * C::KTILE;
    for (int c = 0; c < C::PANELS; ++c)
      tma_load_2d(dst + c * C::KPANEL, is_v ? &tmv : &tmk, full, hk * D + c * C::PCOLS, int(k0) + (t0 + j) * KEYS);
  };
  constexpr int AHEAD = C::VS / 2;

  if (threadIdx.x == 0) {
    prefetch_tmap(&tmq);
    prefetch_tmap(&tmk);
    prefetch_tmap(&tmv);
    mbar_init(q_full, 1);
    for (int g = 0; g < 2; ++g) {
      mbar_init(&s_full[g], 1);
      mbar_init(&p_full[2 * g], 128);
      mbar_init(&p_full[2 * g + 1], 128);
      mbar_init(&o_full[g], 1);
    }
    mbar_init(drain, 1);
    for (int i = 0; i < C::KS; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
    }
    for (int i = 0; i < C::VS; ++i) {
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
      mbar_init(&v_clear[i], 1);
    }
    mbar_init(v_tail, 1);
    *abort_flag = 0;
    fence_barrier_init();
    // the first loads, while the other warps come up
    if (nkt > 0) {
      const int tiles = pair ? 2 : 1;
      mbar_arrive_expect_tx(q_full, tiles * C::PANELS * qpt * G * C::ROWB);
      for (int g = 0; g < tiles; ++g)
        for (int c = 0; c < C::PANELS; ++c)
          tma_load_3d(sQ + g * C::QTILE + c * C::QPANEL, &tmq, q_full, c * C::PCOLS, hk * G, int(q0) + qb + g * qpt);
      for (int j = 0; j <= AHEAD; ++j) {
        if (j < nkt) load_tile(j, false);
        if (j < AHEAD && j < nkt) load_tile(j, true);
      }
    }
  }
  if (warp == 1) tmem_alloc(tmem_holder, C::COLS);
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  const uint32_t tmem = *tmem_holder;
  auto wwait = [&](uint64_t* bar, uint32_t parity, int code) -> bool {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, code));
  };

  if (warp < C::FIRST) {
    if (C::ONE) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::REGS_ISSUE));
    if (warp == 0 && nkt > 0) {
      uint32_t pend_k = 0, pend_v = 0;  // last issued parity per ring slot (bit 1: issued)
      for (int j = 0; j <= AHEAD && j < nkt; ++j) {
        pend_k |= 2u << (2 * j);
        if (j < AHEAD) pend_v |= 2u << (2 * j);
      }
      auto load = [&](int j, bool is_v) -> bool {
        if (j >= nkt) return true;
        const int st = is_v ? j % C::VS : j % C::KS;
        const uint32_t u = uint32_t(is_v ? j / C::VS : j / C::KS) & 1;
        if (!wwait(is_v ? &v_empty[st] : &k_empty[st], u ^ 1, is_v ? 102 : 101)) return false;
        if (lane == 0) load_tile(j, is_v);
        __syncwarp();
        uint32_t& pend = is_v ? pend_v : pend_k;
        pend = (pend & ~(3u << (2 * st))) | ((2u | u) << (2 * st));
        return true;
      };
      // mask values of a tile's states, lane by lane (0 past the end), loaded a tile ahead
      float mk[KEYS / 32];
      auto load_mask = [&](int j) {
#pragma unroll
        for (int i = 0; i < KEYS / 32; ++i) {
          const int jj = (t0 + j) * KEYS + 32 * i + lane;
          mk[i] = jj < nk ? (p.mask ? __ldg(p.mask + k0 + jj) : 1.f) : 0.f;
        }
      };
      // Tile j's rows are looked at before V of tile j + AHEAD is loaded, whose slot is free once the product
      // of tile j - AHEAD is done: the clearing runs ahead of the products.
      bool ok = true;
      if (p.mask) load_mask(0);
      for (int j = 0; j < nkt && ok; ok = ok && load(j + AHEAD + 1, false) && load(j + AHEAD, true), ++j) {
        if (!p.mask && (t0 + j + 1) * KEYS <= nk) continue;
        if (!p.mask) load_mask(j);
        const int st = j % C::VS;
        uint32_t dropped = 0;  // bit i: state 32 i + lane of the tile
#pragma unroll
        for (int i = 0; i < KEYS / 32; ++i) dropped |= mk[i] > 0.5f ? 0u : 1u << i;
        if (p.mask) load_mask(j + 1);
        if (__any_sync(0xffffffffu, dropped != 0)) {
          ok = wwait(&v_full[st], uint32_t(j / C::VS) & 1, 112);
          if (!ok) break;
          // a lane clears its own rows, starting at a piece of its own so that the lanes spread over the banks
          constexpr int PIECES = C::ROWB / 16;
#pragma unroll
          for (int i = 0; i < KEYS / 32; ++i)
            if ((dropped >> i) & 1u) {
              uint8_t* row = sV + st * C::KTILE + (32 * i + lane) * C::ROWB;
#pragma unroll
              for (int e = 0; e < PIECES * C::PANELS; ++e)
                *reinterpret_cast<uint4*>(row + e / PIECES * C::KPANEL + ((e + lane) % PIECES) * 16) = make_uint4(0, 0, 0, 0);
            }
          fence_proxy_async_smem();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(p.mask ? &v_clear[st] : v_tail);
      }
      if (!ok) {
        // every copy this warp issued lands before the CTA ends
        *abort_flag = 1;
        mbar_wait(q_full, 0, 103);
        for (int i = 0; i < C::KS; ++i)
          if ((pend_k >> (2 * i)) & 2u) mbar_wait(&k_full[i], (pend_k >> (2 * i)) & 1u, 104);
        for (int i = 0; i < C::VS; ++i)
          if ((pend_v >> (2 * i)) & 2u) mbar_wait(&v_full[i], (pend_v >> (2 * i)) & 1u, 105);
      }
    }
    if (warp == 1 && nkt > 0) {  // all lanes in step, one issues
      const uint32_t idesc_s = idesc_f16(128, KEYS);
      const uint32_t idesc_o = idesc_f16(128, D) | (1u << 16);  // V MN-major
      const bool lead = elect_one();
      // Tile `it` of stream g: tile `it` of the split in a pair, else 2 it + g. A ring stage is waited for by
      // its first product and freed behind its last (stream 1's in a pair).
      const uint64_t dq0 = tile_desc<D>(sQ), dk0 = tile_desc<D>(sK), dv0 = tile_desc<D>(sV);
      constexpr uint64_t Q16 = uint64_t(C::QTILE >> 4), K16 = uint64_t(C::KTILE >> 4);
      const bool ragged = (t0 + nkt) * KEYS > nk;  // the last tile has states past the end
      int ks = 0, vs = 0;       // ring stages of the next K and V tile
      uint32_t kp = 0, vp = 0;  // and their parities
      auto issue_s = [&](int g) -> bool {
        if (!pair || g == 0) {
          if (!wwait(&k_full[ks], kp, 106)) return false;
          fence_after_sync();
        }
        const uint64_t dq = dq0 + (pair && g ? Q16 : 0ull), dk = dk0 + ks * K16;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const int panel = k / (C::PCOLS / 16), step = k % (C::PCOLS / 16);
          mma_f16_if(lead, tmem + uint32_t(g) * C::S_STRIDE, dq + uint64_t(panel * (C::QPANEL >> 4) + step * 2),
                     dk + uint64_t(panel * (C::KPANEL >> 4) + step * 2), idesc_s, k ? 1u : 0u);
        }
        mma_commit_if(lead, &s_full[g]);
        if (!pair || g == 1) {
          mma_commit_if(lead, &k_empty[ks]);
          if (++ks == C::KS) {
            ks = 0;
            kp ^= 1;
          }
        }
        return true;
      };
      auto issue_o = [&](int g, int it, bool last) -> bool {
        if (!pair || g == 0) {
          if (!wwait(&v_full[vs], vp, 109)) return false;
          if (p.mask ? !wwait(&v_clear[vs], vp, 114) : (ragged && (pair ? it : 2 * it + g) == nkt - 1 && !wwait(v_tail, 0, 115)))
            return false;
        }
        const uint64_t dv = dv0 + vs * K16;
        const uint32_t pa = tmem + uint32_t(g) * C::S_STRIDE, oa = tmem + C::O_COL + uint32_t(g * D);
#pragma unroll
        for (int k = 0; k < KEYS / 16; ++k) {
          if (k % (KEYS / 16 / C::HALVES) == 0) {
            if (!wwait(&p_full[2 * g + (k ? 1 : 0)], uint32_t(it) & 1, 108)) return false;
            fence_after_sync();
          }
          mma_f16_ts_if(lead, oa, pa + uint32_t(8 * k), dv + uint64_t(k * ((16 * C::ROWB) >> 4)), idesc_o, (it || k) ? 1u : 0u);
        }
        if (last) mma_commit_if(lead, &o_full[g]);
        if (!pair || g == 1) {
          mma_commit_if(lead, &v_empty[vs]);
          if (++vs == C::VS) {
            vs = 0;
            vp ^= 1;
          }
        }
        return true;
      };
      bool ok = wwait(q_full, 0, 107) && issue_s(0) && (n1_of == 0 || issue_s(1));
      for (int it = 0; it < n0_of && ok; ++it) {
        const bool two = it < n1_of, next0 = it + 1 < n0_of, next1 = it + 1 < n1_of;
        ok = issue_o(0, it, !next0);
        if (next0) ok = ok && issue_s(0);
        if (two) ok = ok && issue_o(1, it, !next1);
        if (next1) ok = ok && issue_s(1);
      }
      if (!ok) {
        *abort_flag = 1;
        if (lead) mma_commit(drain);
        __syncwarp();
        mbar_wait(drain, 0, 110);
      }
    }
  } else {
    if (C::ONE) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::REGS_SOFTMAX));
    const int g = (warp - C::FIRST) >> 2;
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;  // row of the tile = TMEM lane
    const uint32_t trow = tmem + (uint32_t(quarter * 32) << 16);
    const uint32_t s_addr = trow + uint32_t(g) * C::S_STRIDE, o_addr = trow + C::O_COL + uint32_t(g * D);
    const int n_mine = g ? n1_of : n0_of;
    const float* mb = p.mask ? p.mask + k0 : nullptr;
    bool ok = true;
    constexpr int W = KEYS / 32;  // words of a tile's states
    // mask values of a tile's states, lane by lane (0 past the end), loaded a tile ahead
    float mk[W];
    auto load_mask = [&](int it) {
      const int first = (t0 + (pair ? it : 2 * it + g)) * KEYS;
#pragma unroll
      for (int c = 0; c < W; ++c) {
        const int jj = first + 32 * c + lane;
        mk[c] = it < n_mine && jj < nk ? __ldg(mb + jj) : 0.f;
      }
    };
    if (mb) load_mask(0);
    float m = -INFINITY, l = 0.f;
    for (int it = 0; it < n_mine; ++it) {
      const int j = pair ? it : 2 * it + g;
      const int left = nk - (t0 + j) * KEYS;
      // a tile with states to drop: which are kept, as bits (the same for every row)
      uint32_t km[W];
      bool whole = left >= KEYS;
      if (mb) {
        uint32_t every = 0xffffffffu;
#pragma unroll
        for (int c = 0; c < W; ++c) {
          km[c] = __ballot_sync(0xffffffffu, mk[c] > 0.5f);
          every &= km[c];
        }
        whole = every == 0xffffffffu;
        load_mask(it + 1);
      } else if (!whole) {
#pragma unroll
        for (int c = 0; c < W; ++c) {
          const int n = left - 32 * c;
          km[c] = n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u;
        }
      }
      if (!wwait(&s_full[g], uint32_t(it) & 1, 111)) { ok = false; break; }
      fence_after_sync();
      uint32_t sr[W][32];
#pragma unroll
      for (int c = 0; c < W; ++c) tmem_ld32(s_addr + 32 * c, sr[c]);
      tmem_ld_wait();
#pragma unroll
      for (int c = 0; c < W; ++c) settle(sr[c]);
      if (!whole) {
#pragma unroll
        for (int c = 0; c < W; ++c)
#pragma unroll
          for (int i = 0; i < 32; ++i) sr[c][i] = (km[c] >> i) & 1u ? sr[c][i] : 0xFF800000u;
      }
      float mr[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < W; ++c)
#pragma unroll
        for (int i = 0; i < 32; i += 2)
          mr[(i >> 1) & 3] = fmax3(mr[(i >> 1) & 3], __uint_as_float(sr[c][i]), __uint_as_float(sr[c][i + 1]));
      const float cand = fmaxf(fmaxf(mr[0], mr[1]), fmaxf(mr[2], mr[3])) * p.scale_log2;
      const bool moves = cand - m > RISE;  // (also the first kept state: m = -inf)
      if (__any_sync(0xffffffffu, moves)) {
        const float corr = moves ? ex2_approx(m - cand) : 1.f;
        if (moves) m = cand;
        l *= corr;
        if (it > 0) {
          // the products before this S are done: O may be rescaled
#pragma unroll 1
          for (int c = 0; c < D; c += 16) {
            uint32_t o[16];
            tmem_ld16(o_addr + c, o);
            tmem_ld_wait();
            settle(o);
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
            tmem_st16(o_addr + c, o);
          }
          tmem_st_wait();
        }
      }
      float ref = m == -INFINITY ? 0.f : m - LIFT;
      // 2^(s scale - m) in one step keeps the bits of the product that m, the rounded one, lacks: up to half a
      // unit of m in the last place, far outside f16 for the largest. There the products of the row are rounded
      // first, and the exponents taken back to the scale of scores (a factor of the row's own instead takes a
      // register that the others lack: 5 % slower).
      const bool far = fabsf(ref) > EXACT_REF;
      if (__any_sync(0xffffffffu, far)) {
        const float back = 1.f / p.scale_log2;
#pragma unroll
        for (int c = 0; c < W; ++c)
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const float s = __uint_as_float(sr[c][i]);
            sr[c][i] = __float_as_uint(far ? (__fmul_rn(s, p.scale_log2) - ref) * back : s);
          }
        if (far) ref = 0.f;
      }
      float2 ls[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
      constexpr int CHUNK = C::ONE ? 32 : 8;  // packed pairs stored at a time, as the registers allow
#pragma unroll
      for (int c = 0; c < KEYS / 2; c += CHUNK) {
        uint32_t pk[CHUNK];
#pragma unroll
        for (int i = 0; i < CHUNK; ++i) {
          const int k = 2 * (c + i);
          const float2 x = ffma2(make_float2(__uint_as_float(sr[k / 32][k & 31]), __uint_as_float(sr[k / 32][(k + 1) & 31])),
                                 twice(p.scale_log2), twice(-ref));
          const float2 e = make_float2(ex2_approx(x.x), ex2_approx(x.y));
          ls[i & 1] = fadd2(ls[i & 1], e);
          pk[i] = pack_half2(e.x, e.y);
        }
        if constexpr (C::ONE) tmem_st32(s_addr + c, pk);
        else tmem_st8(s_addr + c, pk);
        if ((c + CHUNK) % (KEYS / 2 / C::HALVES) == 0) {
          tmem_st_wait();
          fence_before_sync();
          mbar_arrive(&p_full[2 * g + (c + CHUNK == KEYS / 2 ? C::HALVES - 1 : 0)]);
        }
      }
      l += (ls[0].x + ls[0].y) + (ls[1].x + ls[1].y);
    }
    if (ok && n_mine > 0) {
      ok = wwait(&o_full[g], 0, 113);
      fence_after_sync();
    }
    // this row's share of the output: in a pair the stream's own O; else the two streams' parts, of
    // which stream g's thread writes the columns [g D / 2, (g + 1) D / 2)
    const int qi = qb + (pair ? g * qpt : 0) + r / G, h = hk * G + r % G;
    const bool mine = r < qpt * G && qi < nq;
    float m_out = m, l_out = l, f0 = 1.f, f1 = 0.f;
    if (!pair) {
      float* xm = reinterpret_cast<float*>(sQ + C::QTILE);
      float* xl = xm + 256;
      xm[g * 128 + r] = m;
      xl[g * 128 + r] = l;
      fence_before_sync();
      if (quarter_any(quarter, !ok)) ok = false;
      fence_after_sync();
      const float m0 = xm[r], m1 = xm[128 + r];
      m_out = fmaxf(m0, m1);
      f0 = m0 == -INFINITY ? 0.f : ex2_approx(m0 - m_out);
      f1 = m1 == -INFINITY ? 0.f : ex2_approx(m1 - m_out);
      l_out = f0 * xl[r] + f1 * xl[128 + r];
    } else if (m == -INFINITY) {
      f0 = 0.f;
    }
    if (ok) {
      const bool direct = p.nsplit == 1;
      const int64_t at = mine && !direct ? part_index(p, split, s, qi, h) : 0;
      const float inv = direct ? (l_out == 0.f ? 0.f : 1.f / l_out) : 1.f;
      const int c_begin = pair ? 0 : g * (D / 2), c_end = pair ? D : c_begin + D / 2;
      const uint32_t o0 = trow + C::O_COL + (pair ? uint32_t(g * D) : 0u);
#pragma unroll 1
      for (int c = c_begin; c < c_end; c += 16) {
        uint32_t a[16], b[16];
        // TMEM of a stream without items was never written: its factor is 0 and it is not read
        if ((pair ? n_mine : n0_of) > 0) tmem_ld16(o0 + c, a);
        if (!pair && n1_of > 0) tmem_ld16(o0 + D + c, b);
        tmem_ld_wait();
        settle(a);
        settle(b);
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i)
          v[i] = ((f0 != 0.f ? __uint_as_float(a[i]) * f0 : 0.f) + (f1 != 0.f ? __uint_as_float(b[i]) * f1 : 0.f)) * inv;
        if (!mine) continue;
        if (direct) {
          __half* dst = p.out + (q0 + qi) * p.out_stride + h * D + c;
          uint32_t u[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) u[i] = pack_half2(v[2 * i], v[2 * i + 1]);
          if (p.wide) {
            store_32(dst, u);
          } else {
            reinterpret_cast<uint4*>(dst)[0] = make_uint4(u[0], u[1], u[2], u[3]);
            reinterpret_cast<uint4*>(dst)[1] = make_uint4(u[4], u[5], u[6], u[7]);
          }
        } else {
          uint32_t u[2][8];
#pragma unroll
          for (int i = 0; i < 16; ++i) u[i / 8][i % 8] = __float_as_uint(v[i]);
          store_32(p.part_o + at * D + c, u[0]);
          store_32(p.part_o + at * D + c + 8, u[1]);
        }
      }
      if (mine && !direct && (pair || g == 0)) p.part_ml[at] = make_float2(m_out, l_out);
    } else {
      *abort_flag = 1;
    }
  }
  fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    fence_after_sync();
    tmem_free(tmem, C::COLS);
  }
}

// ---- host side ----

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

// One m16 block of rows to a key head: the kernel whose warps stream k and v through rings of their own.
bool takes_rows_kernel(const kh_cross_attention_args& a) {
  return int64_t(a.max_q) * (a.q_heads / a.kv_heads) <= 16;
}

constexpr int SMS = 148;  // of a B200: the split must not depend on the device the size is asked on

// Row tiles of a CTA of the tile kernel: two where a CTA's time is mostly its start and end (60 sequences of
// 400-600 queries, 12 heads of 64: on 64 states 46 us against 58 with one, on 256 71 against 82; on 512
// equal, on 1,024 57 against 51). With heads of 128, one CTA to an SM, always.
int row_tiles(const kh_cross_attention_args& a) { return a.head_dim == 128 || a.max_k <= 256 ? 2 : 1; }

// CTAs that a sequence's states are split over: as many as fill the SMs (four CTAs each of the rows
// kernel, one or two of the tile kernel), each with enough states to pay for the join.
int splits(const kh_cross_attention_args& a) {
  const int64_t G = a.q_heads / a.kv_heads;
  const bool few = takes_rows_kernel(a);
  const int64_t cta_rows = row_tiles(a) * (TROWS / G);
  const int64_t blocks = few ? 1 : (a.max_q + cta_rows - 1) / cta_rows;
  const int64_t ctas = std::max<int64_t>(1, blocks * a.kv_heads * a.n_seqs);
  const int64_t want = (few ? 4 * SMS : a.head_dim == 128 ? SMS : 2 * SMS) / ctas;
  const int64_t most = few ? a.max_k / 256 : a.max_k / 512;
  return int(std::min<int64_t>(std::max<int64_t>(1, std::min(want, most)), 64));
}

int64_t round256(int64_t n) { return (n + 255) / 256 * 256; }

template <int D, int RW>
void launch_rows(const CUtensorMap& tk, const CUtensorMap& tv, const CrossParams& p, cudaStream_t st) {
  static std::atomic<uint64_t> configured{0};
  once_per_device(configured, [] {
    KH_CUDA(cudaFuncSetAttribute(cross_rows_kernel<D, RW>, cudaFuncAttributeMaxDynamicSharedMemorySize, RCfg<D, RW>::SMEM));
  });
  cross_rows_kernel<D, RW><<<dim3(p.nsplit, p.kv_heads, p.n_seqs), RW * 32, RCfg<D, RW>::SMEM, st>>>(tk, tv, p);
}

constexpr int64_t JOIN_ROWS = 1024;  // from here on a warp to a row (8 rows, 64 splits: 52 us, 62 with a warp)

template <int D, int ROW_TILES>
void launch_tiles(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const CrossParams& p, cudaStream_t st) {
  using C = TCfg<D>;
  static std::atomic<uint64_t> configured{0};
  once_per_device(configured, [] {
    KH_CUDA(cudaFuncSetAttribute(cross_tile_kernel<D, ROW_TILES>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
  });
  const int rows = ROW_TILES * (TROWS / p.G);
  // (no sequence has more queries than the buffer has rows, however generous max_q is)
  const int64_t most = std::min<int64_t>(p.max_q, p.q_rows);
  const dim3 grid(unsigned((most + rows - 1) / rows), unsigned(p.kv_heads * p.nsplit), unsigned(p.n_seqs));
  cross_tile_kernel<D, ROW_TILES><<<grid, C::THREADS, C::SMEM, st>>>(tq, tk, tv, p);
}

template <int D>
void launch(const CrossParams& p, const kh_cross_attention_args& a, bool states, cudaStream_t st) {
  CUtensorMap tk, tv;
  auto state_maps = [&](int box_cols, int box_rows, int row_bytes) {
    const uint64_t cols = uint64_t(a.kv_heads) * D;
    encode_tensor_map_f16(&tk, a.k, uint64_t(a.kv_rows), cols, uint64_t(a.k_stride), uint32_t(box_cols), uint32_t(box_rows), row_bytes);
    encode_tensor_map_f16(&tv, a.v, uint64_t(a.kv_rows), cols, uint64_t(a.v_stride), uint32_t(box_cols), uint32_t(box_rows), row_bytes);
  };
  if (takes_rows_kernel(a)) {
    // (without states no map is read; any valid one will do)
    using C = RCfg<D, 4>;
    if (states) state_maps(C::PCOLS, RSTEP, C::ROWB);
    else {
      encode_tensor_map_f16(&tk, a.q, uint64_t(a.q_rows), uint64_t(a.q_heads) * D, uint64_t(a.q_stride), C::PCOLS, RSTEP, C::ROWB);
      tv = tk;
    }
    // Few CTAs are over soonest with four warps each (one request, 12 heads, 128 states: 3.6 us against
    // 4.5 with two); many, that run one after another on an SM, with two (64 requests, 12 heads, 200-512
    // states: 17.5 us against 20.6).
    const bool many = int64_t(p.n_seqs) * p.kv_heads * p.nsplit >= 2 * SMS;
    if (many) launch_rows<D, 2>(tk, tv, p, st);
    else launch_rows<D, 4>(tk, tv, p, st);
  } else {
    using C = TCfg<D>;
    const int qpt = TROWS / p.G;
    CUtensorMap tq;
    encode_tensor_map_f16_3d(&tq, a.q, {uint64_t(D), uint64_t(a.q_heads), uint64_t(a.q_rows)}, D, uint64_t(a.q_stride),
                             {uint32_t(C::PCOLS), uint32_t(p.G), uint32_t(qpt)}, C::ROWB);
    if (states) state_maps(C::PCOLS, C::KEYS, C::ROWB);
    else tk = tv = tq;
    if constexpr (D == 128) launch_tiles<D, 2>(tq, tk, tv, p, st);
    else if (row_tiles(a) == 2) launch_tiles<D, 2>(tq, tk, tv, p, st);
    else launch_tiles<D, 1>(tq, tk, tv, p, st);
  }
  KH_CUDA(cudaGetLastError());
  if (p.nsplit > 1) {
    const int64_t rows = int64_t(p.n_seqs) * p.max_q * p.q_heads;
    const bool many = rows > JOIN_ROWS;
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(many ? (rows + 3) / 4 : rows), 1, 1);
    cfg.blockDim = dim3(128, 1, 1);
    cfg.stream = st;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    KH_CUDA(cudaLaunchKernelEx(&cfg, many ? cross_join_kernel<D, 1> : cross_join_kernel<D, 4>, p, rows));
  }
}

}  // namespace

int64_t cross_attention_workspace(const kh_cross_attention_args* args) {
  check_sizes("kh_cross_attention_f16_workspace", args);
  const int n = splits(*args);
  if (n == 1) return 0;
  const int64_t parts = int64_t(n) * args->n_seqs * args->max_q * args->q_heads;
  return round256(parts * args->head_dim * 4) + parts * 8;
}

void cross_attention(const kh_cross_attention_args* args, cudaStream_t st) {
  const char* fn = "kh_cross_attention_f16";
  check_sizes(fn, args);
  const kh_cross_attention_args& a = *args;
  check_that(a.scale > 0.f && a.scale <= 1e30f, fn, "scale must be above 0, at most 1e30");
  if (a.n_seqs == 0 || a.max_q == 0 || a.q_rows == 0) return;
  const bool states = a.kv_rows > 0 && a.max_k > 0;
  auto aligned = [](const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15) == 0; };
  check_that(a.q && a.out && a.q_starts && a.k_starts && (!states || (a.k && a.v)), fn, "null pointer argument");
  check_that(aligned(a.q) && aligned(a.out) && aligned(a.k) && aligned(a.v), fn,
             "q, k, v and out must be 16-byte aligned");
  check_that(aligned4(a.key_mask) && aligned4(a.q_starts) && aligned4(a.k_starts), fn,
             "key_mask, q_starts and k_starts must be 4-byte aligned");
  const int64_t qw = int64_t(a.q_heads) * a.head_dim, kw = int64_t(a.kv_heads) * a.head_dim;
  const int64_t lim = int64_t(1) << 31;
  check_that(a.q_stride >= qw && a.out_stride >= qw && a.q_stride < lim && a.out_stride < lim &&
                 (!states || (a.k_stride >= kw && a.v_stride >= kw && a.k_stride < lim && a.v_stride < lim)),
             fn, "a stride is shorter than its rows (or 2^31 and more)");
  check_that(a.q_stride % 8 == 0 && a.out_stride % 8 == 0 && a.k_stride % 8 == 0 && a.v_stride % 8 == 0, fn,
             "strides must be multiples of 8");
  check_that(a.out != a.q || a.out_stride == a.q_stride, fn, "out may be q with the same stride alone");
  check_that(!states || (a.out != a.k && a.out != a.v), fn, "out may not be k or v: every query reads them");
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
  p.G = a.q_heads / a.kv_heads;
  p.max_q = a.max_q;
  p.max_k = a.max_k;
  p.nsplit = splits(a);
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.wide = reinterpret_cast<uintptr_t>(a.out) % 32 == 0 && a.out_stride % 16 == 0;
  if (p.nsplit > 1) {
    const int64_t parts = int64_t(p.nsplit) * a.n_seqs * a.max_q * a.q_heads;
    p.part_o = static_cast<float*>(a.workspace);
    p.part_ml = reinterpret_cast<float2*>(static_cast<char*>(a.workspace) + round256(parts * a.head_dim * 4));
  }
  if (a.head_dim == 32) launch<32>(p, a, states, st);
  else if (a.head_dim == 64) launch<64>(p, a, states, st);
  else launch<128>(p, a, states, st);
}

int* cross_attention_wait_word() {
  void* p = nullptr;
  KH_CUDA(cudaGetSymbolAddress(&p, sm100::kh_tc_error));
  return static_cast<int*>(p);
}

}  // namespace kh
