// 8-bit floating point (e4m3) products with a scale for each block of 128: the number form,
// its quantisers, a routed slot's expert, and the weight-streaming product for few rows.
//
// The form. A row x is cut into blocks of 128 columns (the last one short). Per block, in
// fp32: a = max(max|x|, 2^-100), scale s = a / 448, factor f = 448 / a, q = e4m3(x f) (round
// to nearest even; |x f| <= 448 up to one rounding, which e4m3 rounds back to 448). A NaN or
// an infinity in a block makes the whole block's products NaN: a is a maximum of bit patterns,
// which NaN wins, and inf * 0 is NaN. A weight [N, K] has one scale per 128 x 128 block.
//
// A product is y[m, n] = sum_B sx[m, B] sw[n / 128, B] (sum_{k in B} qx[m, k] qw[n, k]): the
// inner sum runs on tensor cores (products of two e4m3 numbers are exact in fp32), the outer
// one in fp32 registers, once per block.
#pragma once

#include <cuda_fp8.h>

#include "alut_common.cuh"

namespace alut {

constexpr int kFp8Block = 128;
constexpr float kE4m3Max = 448.0f;
constexpr float kFp8AmaxFloor = 7.888609052210118e-31f;  // 2^-100: 448 / a stays finite

__host__ __device__ inline int fp8_blocks(int n) { return (n + kFp8Block - 1) / kFp8Block; }

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
// The block's largest magnitude from the largest bit pattern (NaN patterns are the largest).
__device__ __forceinline__ float fp8_amax(uint32_t bits) {
  const float a = __uint_as_float(bits);
  return a < kFp8AmaxFloor ? kFp8AmaxFloor : a;
}
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  return e4m3x2(a, b) | (e4m3x2(c, d) << 16);
}

// Runtime-typed element access (quantisers' inputs, ragged edges, outputs).
__device__ __forceinline__ void store_any(void* p, int64_t i, float v, int dtype) {
  if (dtype == ALUT_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else if (dtype == ALUT_F16) static_cast<__half*>(p)[i] = __float2half_rn(v);
  else static_cast<float*>(p)[i] = v;
}

// ---- quantisers ------------------------------------------------------------------------------

struct QuantArgs {
  int64_t batch, rows;
  int cols;
  const void* src;
  int64_t src_stride_b, src_stride;  // elements
  uint8_t* out;
  int64_t out_stride_b, out_stride;  // bytes
  float* scale;                       // contiguous [batch][row blocks][column blocks]
  int src_vec, out_vec;               // rows start on 16 bytes, output rows on 8
};

// n / d by a 32-bit division where that holds both (64-bit ones take a microsecond each of a short call).
__device__ __forceinline__ int64_t quant_div(int64_t n, int64_t d) {
  return ((n | d) >> 32) == 0 ? static_cast<uint32_t>(n) / static_cast<uint32_t>(d) : n / d;
}
template <typename TX>
struct F8Raw8 {  // 8 elements as they lie
  uint4 w[sizeof(TX) / 2];
};
template <typename TX>
__device__ __forceinline__ void f8_widen(const F8Raw8<TX>& r, float (&v)[8]) {
  const TX* e = reinterpret_cast<const TX*>(&r);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = to_f32<TX>(e[j]);
}
// 8 columns of a row, zero from `left` on; and their 8-bit form, as many as there are.
template <typename TX>
__device__ __forceinline__ void quant_load8(const TX* p, int64_t left, bool vec, F8Raw8<TX>& v) {
  if (vec && left >= 8) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(TX) / 2); ++i) v.w[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
    return;
  }
  TX* e = reinterpret_cast<TX*>(&v);
#pragma unroll
  for (int j = 0; j < 8; ++j) e[j] = j < left ? p[j] : from_f32<TX>(0.f);
}
__device__ __forceinline__ void quant_store8(uint8_t* p, int64_t left, bool vec, const float (&v)[8], float f) {
  const uint2 q = make_uint2(e4m3x4(v[0] * f, v[1] * f, v[2] * f, v[3] * f), e4m3x4(v[4] * f, v[5] * f, v[6] * f, v[7] * f));
  if (vec && left >= 8) {
    *reinterpret_cast<uint2*>(p) = q;
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < left) p[j] = static_cast<uint8_t>((j < 4 ? q.x : q.y) >> (8 * (j & 3)));
}

// One scale per row and 128 columns. Memory-bound: a warp takes 4 blocks of a row, two side by side (16
// lanes of 8 columns each), all loads before the first maximum. 8192 x 4096 bf16: 30 us (3.3 TB/s); with
// 2 blocks 34, with 8 40; 16 x 4096: 2.2 us, 2.0, 3.2.
constexpr int kQuantBlocks = 4;
template <typename TX>
__global__ void __launch_bounds__(256) k_fp8_quantize_rows(QuantArgs a) {
  const int lane = threadIdx.x & 31, sub = lane & 15, side = lane >> 4;
  const int kb = fp8_blocks(a.cols), chunks = (kb + kQuantBlocks - 1) / kQuantBlocks;
  const int64_t n = a.batch * a.rows * chunks;
  for (int64_t i = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5; i < n;
       i += (static_cast<int64_t>(gridDim.x) * blockDim.x) >> 5) {
    const int64_t row = quant_div(i, chunks), bi = quant_div(row, a.rows), r = row - bi * a.rows;
    const int b0 = static_cast<int>(i - row * chunks) * kQuantBlocks + side;
    const int64_t c0 = static_cast<int64_t>(b0) * kFp8Block + sub * 8;
    const TX* src = static_cast<const TX*>(a.src) + bi * a.src_stride_b + r * a.src_stride + c0;
    uint8_t* out = a.out + bi * a.out_stride_b + r * a.out_stride + c0;
    F8Raw8<TX> raw[kQuantBlocks / 2];
#pragma unroll
    for (int u = 0; u < kQuantBlocks / 2; ++u)
      quant_load8<TX>(src + 2 * u * kFp8Block, a.cols - c0 - 2 * u * kFp8Block, a.src_vec, raw[u]);
#pragma unroll
    for (int u = 0; u < kQuantBlocks / 2; ++u) {
      float v[8];
      f8_widen<TX>(raw[u], v);
      uint32_t m = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) m = max(m, abs_bits(v[j]));
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
      if (b0 + 2 * u >= kb) continue;
      const float am = fp8_amax(m);
      quant_store8(out + 2 * u * kFp8Block, a.cols - c0 - 2 * u * kFp8Block, a.out_vec, v, kE4m3Max / am);
      if (sub == 0) a.scale[row * kb + b0 + 2 * u] = am / kE4m3Max;
    }
  }
}

// One scale per 128 x 128 block (weights): a CTA per block, which stays in registers between its
// maximum and its form. Four CTAs per SM, that some load while others convert: 128 x 1536 x 2048 bf16 423
// us (2.9 TB/s), with two (119 registers, none spilled) 551, with six 679.
template <typename TX>
__global__ void __launch_bounds__(256, sizeof(TX) == 2 ? 4 : 3) k_fp8_quantize_blocks(QuantArgs a) {
  __shared__ uint32_t s_max[2];
  const int kb = fp8_blocks(a.cols);
  const int64_t rb = (a.rows + kFp8Block - 1) / kFp8Block;
  const int64_t n = a.batch * rb * kb;
  constexpr int kU = kFp8Block * kFp8Block / 8 / 256;
  const int c = (threadIdx.x & 15) * 8, rt = threadIdx.x >> 4;  // rows rt, rt + 16, ...
  if (threadIdx.x < 2) s_max[threadIdx.x] = 0;
  __syncthreads();
  int turn = 0;
  for (int64_t i = blockIdx.x; i < n; i += gridDim.x, turn ^= 1) {
    const int64_t br = quant_div(i, kb), bi = quant_div(br, rb), ri = br - bi * rb;
    const int ci = static_cast<int>(i - br * kb);
    const int64_t r0 = ri * kFp8Block;
    const int nr = static_cast<int>(min(static_cast<int64_t>(kFp8Block), a.rows - r0));
    const int nc = min(kFp8Block, a.cols - ci * kFp8Block);
    const TX* src = static_cast<const TX*>(a.src) + bi * a.src_stride_b + r0 * a.src_stride + ci * kFp8Block + c;
    uint8_t* out = a.out + bi * a.out_stride_b + r0 * a.out_stride + ci * kFp8Block + c;
    F8Raw8<TX> raw[kU];
    uint32_t m = 0;
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int r = rt + 16 * u;
      quant_load8<TX>(src + r * a.src_stride, r < nr ? nc - c : 0, a.src_vec, raw[u]);
    }
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      float v[8];
      f8_widen<TX>(raw[u], v);
#pragma unroll
      for (int j = 0; j < 8; ++j) m = max(m, abs_bits(v[j]));
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if ((threadIdx.x & 31) == 0) atomicMax(&s_max[turn], m);
    __syncthreads();
    const float am = fp8_amax(s_max[turn]);
    const float f = kE4m3Max / am;
    if (threadIdx.x == 0) {
      s_max[turn ^ 1] = 0;  // the next block's; read last before this barrier
      a.scale[i] = am / kE4m3Max;
    }
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int r = rt + 16 * u;
      float v[8];
      f8_widen<TX>(raw[u], v);
      if (r < nr) quant_store8(out + r * a.out_stride, nc - c, a.out_vec, v, f);
    }
    __syncthreads();  // (the cleared maximum)
  }
}

// ---- routed slots --------------------------------------------------------------------------------

struct Fp8Route {
  int q, s, e;
  const int64_t* sel;
  int64_t sel_stride;
  const uint8_t* compute;  // NULL: every slot
  int64_t compute_stride;
  int flat;                // sel and compute are contiguous
  uint32_t* err;
};

// The expert of slot i, or -1 if the slot is not computed (or names no expert).
__device__ __forceinline__ int fp8_slot_expert(const Fp8Route& r, int i, bool& bad) {
  int64_t at = i, cat = i;
  if (!r.flat) {  // rows with gaps: the token's row and the slot in it
    const uint32_t t = static_cast<uint32_t>(i) / static_cast<uint32_t>(r.s);
    const int s = i - static_cast<int>(t) * r.s;
    at = t * r.sel_stride + s;
    cat = t * r.compute_stride + s;
  }
  const int64_t e = r.sel[at];  // both loads at once
  if (r.compute && !r.compute[cat]) return -1;
  if (e < 0 || e >= r.e) {
    bad = true;
    return -1;
  }
  return static_cast<int>(e);
}

constexpr int kFp8MaxExperts = 2048;  // two per thread of the plan

// ---- the weight-streaming product ---------------------------------------------------------------
//
// For few rows the time is the weights' way from HBM. A CTA takes 8 rows of x (the N of mma.sync
// m16n8k32, weights as the M operand) and a slice of weight rows, in steps of two 16-row tiles per
// warp, which are the gate and the up rows of 16 hidden units, or 32 adjacent output columns. The
// eight warps are 8 / ks row groups; the ks warps of a group split K by blocks of 128 and add up
// through shared memory in warp order: ks = 8 where few CTAs have to hide the latency of one token,
// less where there are enough (fewer barriers per byte).
// The weights come by 16-byte asynchronous copies into a ring in shared memory, kStreamDepth steps
// ahead: 64 KB in flight per CTA (registers held a quarter of that), two CTAs per SM up to K = 3840
// and one above, where x's words, 1 KB for 128 columns, take the rest. Every lane
// copies the 16 bytes that it reads itself (4 lanes a row, both 64-byte halves of a block), so the
// ring needs no barrier; and since a dot product may be taken in any order of k, those words are used
// as they lie, x's in the same order. x is quantised once per CTA, by the warp that needs the block:
// lane (g, c) holds 32 of row g's 128 columns, four lanes agree on the maximum, the words wait in
// shared memory. Up to 8 routed slots need no plan: an expert's first slot leads.
// Measured, weights from HBM, one row: 2048 x 2048 5.6 us, 4096 x 4096 10.2, 150000 x 2048 58 (5.3
// TB/s); 8 slots of 8 experts of 2048 x 768 (38 MB, two launches) 24.6. The small ones are bound by
// latency: launch, x's form, the first weights, the reduction over warps. With one CTA per SM 4096 x
// 8192 takes 18 us.

constexpr int kStreamRows = 8;        // rows of x per CTA
constexpr int kStreamWRows = 16;      // weight rows per tile, two tiles per step
constexpr int kStreamWarps = 8;
constexpr int kStreamMaxSteps = 3;    // steps per CTA
constexpr int kStreamMaxSlots = 8;    // routed slots of a call (its rule: experts_stream)
static_assert(kStreamMaxSlots <= kStreamRows, "an expert's slots are one CTA's rows");
constexpr int kStreamMaxBlocks = 64;  // of 128 columns: x's words in shared memory take 1 KB each
constexpr int kStreamDepth = 2;       // steps' weights in flight per warp
constexpr int kStreamStepUnits = 8 * 32;  // 16-byte units of a warp's step: [tile][row g, g + 8][64-byte half][lane]
// Shared memory: the ring [warps][depth][units], x's words [block][2][32 lanes] and scales
// [block][8 rows], the weight's scales [steps][row group][tile][block].
__host__ __device__ inline size_t stream_smem_bytes(int k, int steps, int ks) {
  return static_cast<size_t>(kStreamWarps) * kStreamDepth * kStreamStepUnits * sizeof(uint4) +
         static_cast<size_t>(fp8_blocks(k)) * (64 * sizeof(uint4) + (kStreamRows + 2 * steps * (kStreamWarps / ks)) * sizeof(float));
}

enum Fp8Mode { kFp8Linear = 0, kFp8GateUp = 1, kFp8Down = 2 };

struct StreamArgs {
  Fp8Route r;               // GateUp, Down
  const void* x;            // rows of x: m rows (Linear), q tokens (GateUp), slots (Down, fp32)
  int64_t x_stride;
  int x_vec;                // rows can be read 16 bytes at a time
  int m, n, k;              // rows (Linear), weight rows (per half), reduction length
  const uint8_t* w;         // row r of expert e: w + e * w_stride_e + r * w_stride
  int64_t w_stride, w_stride_e, w_stride_half;
  const float* ws;          // scales, contiguous [E][halves][blocks n][blocks k]
  void* out;                // Linear: [m, n]; GateUp: fp32 [slots][n]; Down: [q, s, n]
  int out_dtype;
  int64_t out_stride, out_stride_s;
  int zero_skipped;
  int steps, lks;           // steps per CTA, log2 of the warps that split K
};

// 16 bytes to shared memory, of which the first `bytes` are read and the rest zero.
__device__ __forceinline__ void cp_async16_part(void* dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(dst))),
               "l"(src), "r"(bytes)
               : "memory");
}
// 16 elements of a row of x from column c on, zero from column k on.
// COHERENT: the rows were written by the kernel this one may overlap (not the read-only path).
template <typename TX, bool COHERENT>
__device__ __forceinline__ void x16(const TX* row, int c, int k, bool live, bool vec, float (&v)[16]) {
  if (live && vec && c + 16 <= k) {
    if constexpr (COHERENT) {
      static_assert(sizeof(TX) == 4, "fp32 rows");
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float4 f = __ldcg(reinterpret_cast<const float4*>(row + c) + j);
        v[4 * j] = f.x;
        v[4 * j + 1] = f.y;
        v[4 * j + 2] = f.z;
        v[4 * j + 3] = f.w;
      }
      return;
    }
    float (&lo)[8] = reinterpret_cast<float (&)[8]>(v[0]);
    float (&hi)[8] = reinterpret_cast<float (&)[8]>(v[8]);
    load8<TX>(row + c, lo);
    load8<TX>(row + c + 8, hi);
    return;
  }
#pragma unroll
  for (int j = 0; j < 16; ++j) v[j] = live && c + j < k ? to_f32<TX>(COHERENT ? __ldcg(row + c + j) : row[c + j]) : 0.f;
}
__device__ __forceinline__ void mma_e4m3(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// silu(g) u by the approximate exponential and reciprocal instructions: relative error about (4 + 1.2
// |g|) 2^-23 (for negative g, where exp(-g) counts), far under the e4m3 rounding that follows; with the
// exact ones a tile of the many-row product took 16000 cycles more. exp(-g) = inf gives 0, silu's limit.
constexpr float kLog2E = 1.44269504f;
__device__ __forceinline__ float exp2_approx(float x) {
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(x));
  return x;
}
__device__ __forceinline__ float rcp_approx(float x) {
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(x));
  return x;
}
__device__ __forceinline__ float silu_mul(float g, float u) { return g * rcp_approx(1.0f + exp2_approx(g * -kLog2E)) * u; }

template <typename TX, int MODE>
__global__ void __launch_bounds__(32 * kStreamWarps, 2) k_fp8_stream(StreamArgs a) {
  constexpr unsigned kAll = 0xffffffffu;
  constexpr int kStepRows = MODE == kFp8GateUp ? kStreamWRows : 2 * kStreamWRows;  // of each half
  extern __shared__ uint4 stream_smem[];
  __shared__ float red[2][kStreamWarps][2][kStreamRows][kStreamWRows + 1];  // [parity of the step]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int ks = 1 << a.lks, groups = kStreamWarps >> a.lks;  // of rows
  const int ki = warp & (ks - 1), rg = warp >> a.lks;         // this warp's share of K, its row group
  const int g = lane >> 2, c = lane & 3;
  const int y = blockIdx.x;  // rows: CTAs that share weights run together
  const int slice = blockIdx.y;
  const int kblocks = fp8_blocks(a.k), nblocks = fp8_blocks(a.n);
  uint4* ring = stream_smem + warp * kStreamDepth * kStreamStepUnits + lane;
  uint4* xw = stream_smem + kStreamWarps * kStreamDepth * kStreamStepUnits;  // [kblocks][2][32]
  float* xs = reinterpret_cast<float*>(xw + kblocks * 64);              // [kblocks][8]
  float* sws = xs + kblocks * kStreamRows;                              // [steps][groups][2][kblocks]
  // Only the down product may start early. What follows it may read its results without knowing that
  // they are on their way (the lookups' combine), so the last kernel of a call lets nobody ahead.
  if constexpr (MODE == kFp8GateUp) pdl_launch_dependents();
  // This CTA's rows: lane m < cnt holds the m-th (Linear: row, otherwise slot).
  int cnt, member = 0, expert = 0;
  if constexpr (MODE == kFp8Linear) {
    cnt = min(kStreamRows, a.m - y * kStreamRows);
    member = y * kStreamRows + lane;
  } else {
    const int n = a.r.q * a.r.s;
    bool bad = false;
    const int id = lane < n ? fp8_slot_expert(a.r, lane, bad) : -1;
    if (bad && lane == y && a.r.err && warp == 0 && slice == 0) atomicOr(a.r.err, static_cast<uint32_t>(kErrBadExpert));
    expert = __shfl_sync(kAll, id, y);
    if (expert < 0) {
      if (MODE == kFp8Down && a.zero_skipped) {
        const int64_t o = static_cast<int64_t>(y / a.r.s) * a.out_stride + (y % a.r.s) * a.out_stride_s;
        const int c0 = slice * a.steps * groups * kStepRows, c1 = min(a.n, c0 + a.steps * groups * kStepRows);
        for (int i = c0 + tid; i < c1; i += blockDim.x) store_any(a.out, o + i, 0.f, a.out_dtype);
      }
      return;
    }
    const unsigned hits = __ballot_sync(kAll, id == expert);
    if (hits & ((1u << y) - 1u)) return;  // an expert's first slot leads
    cnt = __popc(hits);
    if (lane < cnt) member = __fns(hits, 0, lane + 1);
  }
  const int all = groups * kStepRows;  // rows of a step
  const int r0 = slice * a.steps * all;
  const int steps = min(a.steps, (a.n - r0 + all - 1) / all);
  const int mykb = (kblocks - ki + ks - 1) >> a.lks;  // k-blocks ki, ki + ks, ...
  const int row0 = r0 + rg * kStepRows;           // this warp's first rows
  const uint8_t* wbase = a.w + expert * a.w_stride_e + static_cast<int64_t>(row0 + g) * a.w_stride + 16 * c;
  const int64_t tile_stride = MODE == kFp8GateUp ? a.w_stride_half : kStreamWRows * a.w_stride;
  // Every row and column of the slice is there: no copy needs to look.
  const bool whole = (a.k & (kFp8Block - 1)) == 0 && r0 + steps * all <= a.n;
  int istep = 0, ij = 0;  // the next to issue: for each step's rows, this warp's k-blocks
  const uint8_t* ip = wbase + ki * kFp8Block;
  const int64_t high = 8 * a.w_stride, next_kb = static_cast<int64_t>(ks) * kFp8Block;
  const int64_t next_step = static_cast<int64_t>(all) * a.w_stride - (mykb - 1) * next_kb;
  auto issue_next = [&](int stage) {
    if (istep < steps) {
      uint4* dst = ring + stage * kStreamStepUnits;
      if (whole) {
        const uint8_t* src = ip;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          cp_async16(dst + (i * 4) * 32, src);
          cp_async16(dst + (i * 4 + 1) * 32, src + 64);
          cp_async16(dst + (i * 4 + 2) * 32, src + high);
          cp_async16(dst + (i * 4 + 3) * 32, src + high + 64);
          src += tile_stride;
        }
      } else {
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const int i = u >> 2, h = (u >> 1) & 1, j = u & 1;
          const int row = row0 + istep * all + (MODE == kFp8GateUp ? 0 : i * kStreamWRows) + 8 * h + g;
          const int bytes = row < a.n ? max(0, min(16, a.k - ((ki + ij * ks) * kFp8Block + 16 * c + 64 * j))) : 0;
          cp_async16_part(dst + u * 32, bytes > 0 ? ip + i * tile_stride + h * high + 64 * j : a.w, bytes);
        }
      }
      if (++ij == mykb) {
        ij = 0;
        ++istep;
        ip += next_step;
      } else {
        ip += next_kb;
      }
    }
    cp_async_commit();  // one group per step, empty behind the last
  };
#pragma unroll
  for (int i = 0; i < kStreamDepth; ++i) issue_next(i);
  for (int st = warp; st < steps * groups * 2; st += kStreamWarps) {  // (step, row group, tile)
    const int t = st & 1;
    const int row = r0 + (st >> 1) * kStepRows + (MODE == kFp8GateUp ? 0 : t * kStreamWRows);
    const int nb = min(row / kFp8Block, nblocks - 1);
    const int64_t half = MODE == kFp8GateUp ? 2 * static_cast<int64_t>(expert) + t : expert;
    for (int kb = lane; kb < kblocks; kb += 32) sws[st * kblocks + kb] = __ldg(a.ws + (half * nblocks + nb) * kblocks + kb);
  }
  if constexpr (MODE == kFp8Down) pdl_wait();  // the weights are on their way meanwhile
  {  // x's 8-bit form, a k-block per warp at a time
    const int src = __shfl_sync(kAll, member, g);
    const TX* xrow = static_cast<const TX*>(a.x) + static_cast<int64_t>(MODE == kFp8GateUp ? src / a.r.s : src) * a.x_stride;
    const bool live = g < cnt;
    for (int kb = warp; kb < kblocks; kb += kStreamWarps) {
      const int c0 = kb * kFp8Block + 16 * c;
      float xv[2][16];
      x16<TX, MODE == kFp8Down>(xrow, c0, a.k, live, a.x_vec, xv[0]);
      x16<TX, MODE == kFp8Down>(xrow, c0 + 64, a.k, live, a.x_vec, xv[1]);
      uint32_t m = 0;
#pragma unroll
      for (int j = 0; j < 16; ++j) m = max(m, max(abs_bits(xv[0][j]), abs_bits(xv[1][j])));
      m = max(m, __shfl_xor_sync(kAll, m, 1));
      m = max(m, __shfl_xor_sync(kAll, m, 2));
      const float am = fp8_amax(m);
      const float f = kE4m3Max / am;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint32_t q[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          q[i] = e4m3x4(xv[j][4 * i] * f, xv[j][4 * i + 1] * f, xv[j][4 * i + 2] * f, xv[j][4 * i + 3] * f);
        xw[(kb * 2 + j) * 32 + lane] = make_uint4(q[0], q[1], q[2], q[3]);
      }
      if (c == 0) xs[kb * kStreamRows + g] = am / kE4m3Max;
    }
  }
  __syncthreads();
  int stage = 0;
  for (int step = 0; step < steps; ++step) {
    float acc[2][4] = {};
    for (int j = 0; j < mykb; ++j) {
      const int kb = ki + j * ks;
      cp_async_wait<kStreamDepth - 1>();
      const uint4* w = ring + stage * kStreamStepUnits;
      const uint4 x0 = xw[kb * 64 + lane], x1 = xw[kb * 64 + 32 + lane];
      const float2 sx = *reinterpret_cast<const float2*>(xs + kb * kStreamRows + 2 * c);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint4 a0 = w[i * 128], a1 = w[i * 128 + 32], b0 = w[i * 128 + 64], b1 = w[i * 128 + 96];
        float d[4] = {};
        mma_e4m3(d, a0.x, b0.x, a0.y, b0.y, x0.x, x0.y);
        mma_e4m3(d, a0.z, b0.z, a0.w, b0.w, x0.z, x0.w);
        mma_e4m3(d, a1.x, b1.x, a1.y, b1.y, x1.x, x1.y);
        mma_e4m3(d, a1.z, b1.z, a1.w, b1.w, x1.z, x1.w);
        const float sw = sws[((step * groups + rg) * 2 + i) * kblocks + kb];
        acc[i][0] = fmaf(d[0], sx.x * sw, acc[i][0]);
        acc[i][1] = fmaf(d[1], sx.y * sw, acc[i][1]);
        acc[i][2] = fmaf(d[2], sx.x * sw, acc[i][2]);
        acc[i][3] = fmaf(d[3], sx.y * sw, acc[i][3]);
      }
      issue_next(stage);  // into the units just used
      if (++stage == kStreamDepth) stage = 0;
    }
    float(&part)[kStreamWarps][2][kStreamRows][kStreamWRows + 1] = red[step & 1];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      part[warp][i][2 * c][g] = acc[i][0];
      part[warp][i][2 * c + 1][g] = acc[i][1];
      part[warp][i][2 * c][g + 8] = acc[i][2];
      part[warp][i][2 * c + 1][g + 8] = acc[i][3];
    }
    __syncthreads();  // (the step after next writes this half again, behind the next step's barrier)
    // Sums over the warps, 16 consecutive columns of a row by 16 consecutive threads. A warp
    // handles whole rows, so that the member comes by a shuffle.
    // (16 rows of a row group's outputs: 8 rows of x, of one or two tiles; the absent are skipped.)
    constexpr int kTiles = MODE == kFp8GateUp ? 1 : 2;
    for (int o0 = warp * 32; o0 < groups * kTiles * kStreamRows * kStreamWRows; o0 += 32 * kStreamWarps) {
      const int o = o0 + lane, col = o & 15;
      const int row = (o >> 4) & 7, i = kTiles == 1 ? 0 : (o >> 7) & 1, og = kTiles == 1 ? o >> 7 : o >> 8;
      const int dst = __shfl_sync(kAll, member, row);
      const int wr = r0 + step * all + og * kStepRows + i * kStreamWRows + col;
      if (row >= cnt || wr >= a.n) continue;
      float v = 0.f, u = 0.f;
      for (int w = og * ks; w < og * ks + ks; ++w) {
        v += part[w][i][row][col];
        if (MODE == kFp8GateUp) u += part[w][1][row][col];
      }
      if constexpr (MODE == kFp8GateUp) {
        static_cast<float*>(a.out)[static_cast<int64_t>(dst) * a.out_stride + wr] = silu_mul(v, u);
      } else if constexpr (MODE == kFp8Down) {
        store_any(a.out, static_cast<int64_t>(dst / a.r.s) * a.out_stride + (dst % a.r.s) * a.out_stride_s + wr, v,
                  a.out_dtype);
      } else {
        store_any(a.out, static_cast<int64_t>(dst) * a.out_stride + wr, v, a.out_dtype);
      }
    }
  }
}

}  // namespace alut
