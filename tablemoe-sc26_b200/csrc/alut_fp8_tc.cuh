// The block-scaled e4m3 product for many rows: tcgen05 (kind::f8f6f4), persistent CTAs.
//
// Tile: 128 rows of x (MMA M) x two 128-row weight blocks (MMA N = 256): adjacent output columns
// (Linear, Down), or the gate and the up rows of the same 128 hidden units (GateUp).
// The scales change with every 128 columns of K, so an accumulator holds one k-block only: the
// MMA of a k-block (4 steps of K = 32) overwrites one of two 128 x 256 fp32 accumulators in
// tensor memory, and the epilogue warps add it, times sx[row, block] sw[block], to fp32 registers
// (128 a thread). Thread r of a column half owns row r, so a k-block has two factors per thread.
// Tensor cores (512 cycles a k-block at the dense e4m3 rate) and epilogue (256 columns of TMEM
// loads and FMAs per lane quarter) run side by side on the two accumulators.
//
//   warps 0-7  epilogue: TMEM lane quarter warp % 4, columns 64 (warp / 4) .. + 64 of each block
//   warp 8     copies: both operands by TMA with the 128-byte swizzle; GateUp gathers x's rows
//              by token (one tile::gather4 of 4 rows per lane and k-block)
//   warp 9     MMA issuer (10, 11 idle: registers are handed over by warpgroups)
//   barriers:  full/empty per stage, full/empty per accumulator
// GateUp ends with h = silu(gate) * up, its 8-bit form (the 128 hidden units of the tile are one
// block of the next product; the two column halves exchange their maxima) written for Down.
// Every wait is bounded in time (error bit, stop, bounded drain, TMEM freed).
#pragma once

#include <cuda.h>

#include "alut_common.cuh"
#include "alut_fp8.cuh"
#include "alut_ptx.cuh"

namespace alut {

constexpr int kF8Rows = 128;
constexpr int kF8Stages = 4;
constexpr uint32_t kF8TileBytes = kF8Rows * kFp8Block;  // one 128 x 128 operand tile
constexpr uint32_t kF8StageBytes = 3 * kF8TileBytes;    // x, two weight blocks
constexpr int kF8EpiWarps = 8;
// Three warpgroups of 128 threads, launched with 168 registers a thread; the epilogue's two need
// more (128 sums, 64 loaded values), the third fewer: 2 x 232 + 40 = 3 x 168.
constexpr int kF8Threads = 32 * (kF8EpiWarps + 4);
constexpr int kF8EpiRegs = 232, kF8RoleRegs = 40;
constexpr int kF8CopyWarp = kF8EpiWarps, kF8MmaWarp = kF8EpiWarps + 1;
constexpr uint32_t kF8TmemCols = 512;
constexpr size_t kF8SmemBytes = 1024 + 1024 + static_cast<size_t>(kF8Stages) * kF8StageBytes;

// Scales of x's rows (and of the hidden rows) are kept [row][blocks rounded up to 4].
__host__ __device__ inline int f8_scale_pitch(int k) { return (fp8_blocks(k) + 3) & ~3; }
__host__ __device__ inline int64_t f8_row_pitch(int k) { return static_cast<int64_t>(fp8_blocks(k)) * kFp8Block; }

struct F8Args {
  int m, n, k;              // rows (Linear), weight rows per half, reduction length
  const float* sx;          // x's scales [rows][f8_scale_pitch(k)]
  const float* ws;          // weight scales, contiguous [E][halves][blocks n][blocks k]
  const int4* groups;       // GateUp, Down: (expert, first position, rows, 0)
  const int* n_groups;
  const int* sorted;        // position -> slot
  int s;                    // slots per token
  uint8_t* hq;              // GateUp: [positions][f8_row_pitch(n)]
  float* hs;                // GateUp: [positions][f8_scale_pitch(n)]
  void* out;                // Linear [m, n], Down [q, s, n]
  int out_dtype, out_vec;   // out_vec: 16-byte stores are aligned
  int64_t out_stride, out_stride_s;
  uint32_t* err;
};

__device__ __forceinline__ void f8_load_tile(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  pt_tma_load_2d(dst, map, x, y, bar);
}
__device__ __forceinline__ void f8_load_weight(void* dst, const CUtensorMap* map, int x, int y, int half, int e,
                                               uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(smem_addr(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(half), "r"(e), "r"(smem_addr(bar))
      : "memory");
}
// Four rows (128 bytes each) of a map whose box is one row high.
__device__ __forceinline__ void f8_gather4(void* dst, const CUtensorMap* map, int x, int4 rows, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, "
      "%4, %5, %6}], [%7];" ::"r"(smem_addr(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(rows.x), "r"(rows.y), "r"(rows.z), "r"(rows.w),
      "r"(smem_addr(bar))
      : "memory");
}
// kind::f8f6f4 instruction descriptor: fp32 D, e4m3 A and B, K-major, M = 128, N = 256.
__host__ __device__ __forceinline__ uint32_t f8_idesc() {
  return (1u << 4) | (static_cast<uint32_t>(256 >> 3) << 17) | (static_cast<uint32_t>(kF8Rows >> 4) << 24);
}
__device__ __forceinline__ void f8_mma(uint32_t tmem, uint64_t da, uint64_t db, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n" ::"r"(
          tmem),
      "l"(da), "l"(db), "r"(idesc), "r"(acc)
      : "memory");
}

// 64 fp32 values as consecutive outputs of a row, columns c .. c + 63 of n.
__device__ __forceinline__ void f8_store64(void* out, int64_t o, const float (&v)[64], int c, int n, int dtype, bool vec) {
  if (vec && c + 64 <= n && dtype != ALUT_F32) {
#pragma unroll
    for (int j = 0; j < 64; j += 8) {
      const float (&w)[8] = reinterpret_cast<const float (&)[8]>(v[j]);
      if (dtype == ALUT_BF16) store8<__nv_bfloat16>(static_cast<__nv_bfloat16*>(out) + o + j, w);
      else store8<__half>(static_cast<__half*>(out) + o + j, w);
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 64; ++j)
    if (c + j < n) store_any(out, o + j, v[j], dtype);
}

template <int MODE>
__global__ void __launch_bounds__(kF8Threads, 1)
    k_fp8_tc(const __grid_constant__ CUtensorMap x_map, const __grid_constant__ CUtensorMap w_map, F8Args a) {
  extern __shared__ unsigned char f8_raw[];
  unsigned char* f8_smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(f8_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(f8_smem);  // [kF8Stages]
  uint64_t* empty = full + kF8Stages;                     // [kF8Stages]
  uint64_t* t_full = empty + kF8Stages;                   // [2]
  uint64_t* t_empty = t_full + 2;                         // [2]
  uint64_t* maxima = t_empty + 2;                         // [1] both column halves' maxima are there
  uint64_t* drain = maxima + 1;                           // [1]
  unsigned char* stages = f8_smem + 1024;                 // [kF8Stages][x | block 0 | block 1]
  __shared__ float s_max[2][2][kF8Rows];                  // [tile parity][column half][row]
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort, s_issued;
  volatile int* abort_flag = &s_abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int kblocks = fp8_blocks(a.k), nblocks = fp8_blocks(a.n);
  pdl_launch_dependents();
  if (warp == kF8MmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&s_tmem)),
                 "r"(kF8TmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (tid == 0) {
    for (int i = 0; i < kF8Stages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&t_full[i], 1);
      mbar_init(&t_empty[i], kF8EpiWarps);
    }
    mbar_init(maxima, kF8EpiWarps);
    mbar_init(drain, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    s_abort = 0;
    s_issued = 0;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  pdl_wait();  // the 8-bit rows, the plan and the scales come from the kernel before
  const int nt = MODE == kFp8GateUp ? nblocks : (nblocks + 1) / 2;  // tiles along the weight rows
  const int mt = MODE == kFp8Linear ? (a.m + kF8Rows - 1) / kF8Rows : __ldcg(a.n_groups);
  const int64_t ntiles = static_cast<int64_t>(mt) * nt;

  if (warp >= kF8EpiWarps) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kF8RoleRegs));
    if (warp == kF8CopyWarp) {
      // ---- copies ------------------------------------------------------------------------------
      int it = 0, st = 0, wrapped = 0;
      bool ok = true;
      for (int64_t tile = blockIdx.x; tile < ntiles && ok; tile += gridDim.x) {
        const int mi = static_cast<int>(tile / nt), ni = static_cast<int>(tile % nt);
        int e = 0, row0 = mi * kF8Rows;
        int4 rows = make_int4(0, 0, 0, 0);
        if constexpr (MODE != kFp8Linear) {
          const int4 g = __ldcg(a.groups + mi);
          e = g.x;
          row0 = g.y;
          if constexpr (MODE == kFp8GateUp) {  // this lane's four rows; rows past the group repeat its first
            int* r = reinterpret_cast<int*>(&rows);
  #pragma unroll
            for (int j = 0; j < 4; ++j) r[j] = __ldcg(a.sorted + g.y + (4 * lane + j < g.z ? 4 * lane + j : 0)) / a.s;
          }
        }
        for (int kb = 0; kb < kblocks; ++kb, ++it, (++st == kF8Stages ? (st = 0, wrapped ^= 1) : 0)) {
          if (lane == 0 && it >= kF8Stages) ok = tc_wait(&empty[st], wrapped ^ 1, abort_flag);
          ok = __shfl_sync(0xffffffffu, ok, 0);
          if (!ok) break;
          unsigned char* sx = stages + static_cast<size_t>(st) * kF8StageBytes;
          if (lane == 0) {
            mbar_expect_tx(&full[st], kF8StageBytes);
            if constexpr (MODE == kFp8GateUp) {
              f8_load_weight(sx + kF8TileBytes, &w_map, kb * kFp8Block, ni * kFp8Block, 0, e, &full[st]);
              f8_load_weight(sx + 2 * kF8TileBytes, &w_map, kb * kFp8Block, ni * kFp8Block, 1, e, &full[st]);
            } else {
              f8_load_tile(sx, &x_map, kb * kFp8Block, row0, &full[st]);
              f8_load_weight(sx + kF8TileBytes, &w_map, kb * kFp8Block, 2 * ni * kFp8Block, 0, e, &full[st]);
              f8_load_weight(sx + 2 * kF8TileBytes, &w_map, kb * kFp8Block, (2 * ni + 1) * kFp8Block, 0, e, &full[st]);
            }
          }
          if constexpr (MODE == kFp8GateUp) {
            __syncwarp();
            f8_gather4(sx + lane * 4 * kFp8Block, &x_map, kb * kFp8Block, rows, &full[st]);
          }
        }
      }
      if (lane == 0) {
        s_issued = it;
        if (!ok && !*abort_flag) {
          *abort_flag = 1;
          if (a.err) atomicOr(a.err, static_cast<uint32_t>(kErrMmaTimeout));
        }
      }
    } else if (warp == kF8MmaWarp) {
      // ---- MMA issuer ----------------------------------------------------------------------------
      if (lane == 0) {
        int it = 0, st = 0, sph = 0;
        bool ok = true;
        const uint32_t idesc = f8_idesc();
        for (int64_t tile = blockIdx.x; tile < ntiles && ok; tile += gridDim.x) {
          for (int kb = 0; kb < kblocks; ++kb, ++it, (++st == kF8Stages ? (st = 0, sph ^= 1) : 0)) {
            const int buf = it & 1;
            if ((it >= 2 && !tc_wait(&t_empty[buf], ((it >> 1) - 1) & 1, abort_flag)) ||
                !tc_wait(&full[st], sph, abort_flag)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t sx = smem_addr(stages + static_cast<size_t>(st) * kF8StageBytes);
  #pragma unroll
            for (int k32 = 0; k32 < kFp8Block / 32; ++k32)
              f8_mma(tmem + buf * 256, pt_desc_sw128(sx + k32 * 32), pt_desc_sw128(sx + kF8TileBytes + k32 * 32), idesc,
                     k32 ? 1u : 0u);
            tc_commit(&empty[st]);
            tc_commit(&t_full[buf]);
          }
        }
        if (!ok && !*abort_flag) {
          *abort_flag = 1;
          if (a.err) atomicOr(a.err, static_cast<uint32_t>(kErrMmaTimeout));
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kF8EpiRegs));
    // ---- epilogue ------------------------------------------------------------------------------
    const int half = warp >> 2;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lane_base = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + half * 64;
    const int pitch = f8_scale_pitch(a.k);
    int it = 0, par = 0;
    bool ok = true;
    auto stop_if = [&](bool bad) {  // whole warps: a wait ran out
      bad = __any_sync(0xffffffffu, bad);
      if (bad && lane == 0 && !*abort_flag) {
        *abort_flag = 1;
        if (a.err) atomicOr(a.err, static_cast<uint32_t>(kErrMmaTimeout));
      }
      return bad;
    };
    for (int64_t tile = blockIdx.x; tile < ntiles && ok; tile += gridDim.x, par ^= 1) {
      const int mi = static_cast<int>(tile / nt), ni = static_cast<int>(tile % nt);
      int e = 0, rows, pos0 = mi * kF8Rows;
      if constexpr (MODE == kFp8Linear) {
        rows = min(kF8Rows, a.m - pos0);
      } else {
        const int4 g = __ldcg(a.groups + mi);
        e = g.x;
        pos0 = g.y;
        rows = g.z;
      }
      const bool live = row < rows;
      int src = pos0 + (live ? row : 0);
      int slot = 0;
      if constexpr (MODE != kFp8Linear) slot = __ldcg(a.sorted + src);
      if constexpr (MODE == kFp8GateUp) src = slot / a.s;
      const float4* sxp = reinterpret_cast<const float4*>(a.sx + static_cast<int64_t>(src) * pitch);
      const int nb0 = MODE == kFp8GateUp ? ni : 2 * ni;
      const float* sw0 = a.ws + ((static_cast<int64_t>(e) * (MODE == kFp8GateUp ? 2 : 1)) * nblocks + nb0) * kblocks;
      // the second block: the up rows' scales, or the next block of columns (none past the last)
      const float* sw1 = MODE == kFp8GateUp ? sw0 + static_cast<int64_t>(nblocks) * kblocks
                                            : (nb0 + 1 < nblocks ? sw0 + kblocks : sw0);
      float acc0[64], acc1[64];
#pragma unroll
      for (int j = 0; j < 64; ++j) acc0[j] = acc1[j] = 0.f;
      float4 s4 = __ldcg(sxp);
      float w0 = __ldg(sw0), w1 = __ldg(sw1);
      for (int kb = 0; kb < kblocks; ++kb, ++it) {
        const int buf = it & 1;
        const float s = (kb & 3) == 0 ? s4.x : (kb & 3) == 1 ? s4.y : (kb & 3) == 2 ? s4.z : s4.w;
        const float f0 = s * w0, f1 = s * w1;
        if (kb + 1 < kblocks) {  // the next block's factors, a k-block ahead
          if (((kb + 1) & 3) == 0) s4 = __ldcg(sxp + ((kb + 1) >> 2));
          w0 = __ldg(sw0 + kb + 1);
          w1 = __ldg(sw1 + kb + 1);
        }
        if (stop_if(!tc_wait(&t_full[buf], (it >> 1) & 1, abort_flag))) {
          ok = false;
          break;
        }
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float v[32];
          tc_ld32(lane_base + buf * 256 + (c >> 1) * 128 + (c & 1) * 32, v);
          if (c == 3) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&t_empty[buf]);
          }
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            if (c < 2) acc0[c * 32 + j] = fmaf(v[j], f0, acc0[c * 32 + j]);
            else acc1[(c - 2) * 32 + j] = fmaf(v[j], f1, acc1[(c - 2) * 32 + j]);
          }
        }
      }
      if (!ok) break;
      if constexpr (MODE == kFp8GateUp) {
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < 64; ++j) {  // columns past I have zero weights: h = 0
          acc0[j] = silu_mul(acc0[j], acc1[j]);
          m = max(m, abs_bits(acc0[j]));
        }
        s_max[par][half][row] = __uint_as_float(m);
        __syncwarp();
        if (lane == 0) mbar_arrive(maxima);
        if (stop_if(!tc_wait(maxima, par, abort_flag))) break;
        m = max(m, __float_as_uint(s_max[par][half ^ 1][row]));
        const float am = fp8_amax(m);
        const float f = kE4m3Max / am;
        if (live) {
          const int64_t pos = pos0 + row;
          uint4* dst = reinterpret_cast<uint4*>(a.hq + pos * f8_row_pitch(a.n) + ni * kFp8Block + half * 64);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint4 q;
            q.x = e4m3x4(acc0[16 * j] * f, acc0[16 * j + 1] * f, acc0[16 * j + 2] * f, acc0[16 * j + 3] * f);
            q.y = e4m3x4(acc0[16 * j + 4] * f, acc0[16 * j + 5] * f, acc0[16 * j + 6] * f, acc0[16 * j + 7] * f);
            q.z = e4m3x4(acc0[16 * j + 8] * f, acc0[16 * j + 9] * f, acc0[16 * j + 10] * f, acc0[16 * j + 11] * f);
            q.w = e4m3x4(acc0[16 * j + 12] * f, acc0[16 * j + 13] * f, acc0[16 * j + 14] * f, acc0[16 * j + 15] * f);
            dst[j] = q;
          }
          if (half == 0) a.hs[pos * f8_scale_pitch(a.n) + ni] = am / kE4m3Max;
        }
      } else if (live) {
        int64_t o;
        if constexpr (MODE == kFp8Linear) o = static_cast<int64_t>(src) * a.out_stride;
        else o = static_cast<int64_t>(slot / a.s) * a.out_stride + static_cast<int64_t>(slot % a.s) * a.out_stride_s;
        const int c = nb0 * kFp8Block + half * 64;
        f8_store64(a.out, o + c, acc0, c, a.n, a.out_dtype, a.out_vec);
        f8_store64(a.out, o + c + kFp8Block, acc1, c + kFp8Block, a.n, a.out_dtype, a.out_vec);
      }
    }
  }

  __syncthreads();
  if (*abort_flag && tid == 32 * kF8MmaWarp) {
    tc_commit(drain);
    mbar_wait_bounded(drain, 0);
  }
  if (*abort_flag && tid == 32 * kF8CopyWarp) {
    const int issued = s_issued;  // copies: the latest use of each stage
    for (int st = 0; st < kF8Stages && st < issued; ++st) {
      const int last = st + ((issued - 1 - st) / kF8Stages) * kF8Stages;
      mbar_wait_bounded(&full[st], (last / kF8Stages) & 1);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kF8MmaWarp)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kF8TmemCols) : "memory");
}

// ---- what the products need first ------------------------------------------------------------

struct F8PrepArgs {
  const void* x;
  int64_t x_stride;
  int rows, k, x_vec;
  uint8_t* xq;  // [rows][f8_row_pitch(k)], columns from k on zero
  float* sx;    // [rows][f8_scale_pitch(k)]
};

// x's 8-bit form: 16 lanes a block of 128 columns, 8 columns a lane.
template <typename TX>
__global__ void __launch_bounds__(256) k_fp8_rows(F8PrepArgs a) {
  pdl_launch_dependents();
  const int kb = fp8_blocks(a.k);
  const int64_t n = static_cast<int64_t>(a.rows) * kb;
  const int sub = threadIdx.x & 15;
  const int64_t step = (static_cast<int64_t>(gridDim.x) * blockDim.x) >> 4;
  for (int64_t i0 = (static_cast<int64_t>(blockIdx.x) * blockDim.x + (threadIdx.x & ~31)) >> 4; i0 < n; i0 += step) {
    const int64_t i = i0 + ((threadIdx.x >> 4) & 1);  // whole warps iterate together (shuffles)
    const bool on = i < n;
    const int64_t row = on ? i / kb : 0;
    const int b = on ? static_cast<int>(i % kb) : 0;
    const int c = b * kFp8Block + sub * 8;
    const TX* src = static_cast<const TX*>(a.x) + row * a.x_stride;
    float v[8];
    if (on && a.x_vec && c + 8 <= a.k) {
      load8<TX>(src + c, v);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = on && c + j < a.k ? to_f32<TX>(src[c + j]) : 0.f;
    }
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, abs_bits(v[j]));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float am = fp8_amax(m);
    const float f = kE4m3Max / am;
    if (on) {
      uint2 q;
      q.x = e4m3x4(v[0] * f, v[1] * f, v[2] * f, v[3] * f);
      q.y = e4m3x4(v[4] * f, v[5] * f, v[6] * f, v[7] * f);
      *reinterpret_cast<uint2*>(a.xq + row * f8_row_pitch(a.k) + c) = q;
      if (sub == 0) a.sx[row * f8_scale_pitch(a.k) + b] = am / kE4m3Max;
    }
  }
}

}  // namespace alut
