// The block-scaled e4m3 product for many rows: tcgen05 (kind::f8f6f4), persistent pairs of CTAs.
//
// Tile of a pair (cta_group::2, one MMA of M = 256, N = 256 over both SMs): 256 rows of x, 128 per
// CTA, x two 128-row weight blocks, adjacent output columns. Each CTA loads its own rows of x and one
// of the two weight blocks: 32 KB per 128 columns of K and CTA. With one CTA per tile it is 48 KB, and
// the copies out of L2 and the operands' way through shared memory (48 KB in, 48 KB out, 128 bytes a
// cycle) set the rate: 1040 cycles a k-block measured against 512 of the tensor cores.
// The scales change with every 128 columns of K, so an accumulator holds one k-block only: the MMAs
// of a k-block (4 steps of K = 32) overwrite it, and the epilogue warps add it, times sx[row, block]
// sw[block], to fp32 registers (128 a thread; a thread owns a row: two factors per k-block). Tensor
// memory holds four accumulators of 128 columns, half a k-block's: the low or high 64 rows of both
// weight blocks (an MMA of N = 128 takes 64 rows from each CTA). What bounds it, measured: the MMAs
// alone 515 cycles a k-block, with the copies 522; but a k-block's MMA is done 950 cycles after its
// issue, and reading it back (128 KB per SM through the TMEM port) takes 540. With two accumulators
// of a whole k-block that chain ran at 1000 cycles a k-block.
//
//   warps 0-7  epilogue: TMEM lane quarter warp % 4; part warp / 4 has one of the two weight blocks
//   warp 8     TMA copies (128-byte swizzle), signalled to the leader CTA's barrier
//   warp 9     MMA issuer (of the pair's leader, rank 0)
//   warp 10    the factors sx sw of a k-block's 128 rows and two blocks, into a ring in shared
//              memory (read by the epilogue itself, their latency cost 460 cycles a k-block)
//   warp 11    waits for the accumulators and lets the epilogue go by a named barrier: of warps
//              that waited on the mbarrier themselves the last woke 600 cycles after the first
//   barriers:  full/empty per stage, full/empty per accumulator, full/empty per ring slot; the
//              stages' full and the accumulators' empty count in the leader, the commits arrive in
//              both CTAs
// A thread ends with a row segment of 128 outputs, which goes out through shared memory so that a
// store instruction writes 256 adjacent bytes of two rows (one bulk copy per row instead took 2400
// cycles a warp to issue).
// Every wait for a copy, an MMA or a factor is bounded in time (error bit, stop, time for what is in
// flight, TMEM freed). The epilogue's named barriers need warp 11 alone, which goes through all of them
// whatever has run out (f8_drain).
// Measured: 8192 x 4096 x 4096 151 us with x's form (23 of them), 1.8 PFLOP/s; 4096 x 4096 x 4096 87; 2048 x
// 2560 x 2560 32. Bound by the accumulators' way back to registers (about 1000 cycles a k-block).
#pragma once

#include <cuda.h>

#include <cooperative_groups.h>

#include "alut_common.cuh"
#include "alut_fp8.cuh"
#include "alut_ptx.cuh"

namespace alut {

constexpr int kF8Rows = 128;                // rows of x per CTA
constexpr int kF8PairRows = 2 * kF8Rows;    // per pair of CTAs
constexpr int kF8Stages = 4;                // of copies: as many as the memory beside the output rows holds
constexpr uint32_t kF8TileBytes = kF8Rows * kFp8Block;  // one 128 x 128 operand tile
constexpr uint32_t kF8StageBytes = 2 * kF8TileBytes;    // x's rows, a weight block
constexpr int kF8EpiWarps = 8;
// Three warpgroups, launched with 168 registers a thread; the epilogue's two need more (128 sums, 64
// loaded values), the third fewer: 2 x 224 + 56 = 3 x 168.
constexpr int kF8Threads = 32 * (kF8EpiWarps + 4);
constexpr int kF8EpiRegs = 224, kF8RoleRegs = 56;
constexpr int kF8CopyWarp = kF8EpiWarps, kF8MmaWarp = kF8EpiWarps + 1, kF8ScaleWarp = kF8EpiWarps + 2, kF8WaitWarp = kF8EpiWarps + 3;
constexpr int kF8Group = 4, kF8Ring = 2;     // factors of 4 k-blocks per ring slot
constexpr uint32_t kF8RowBytes = 256 + 16;    // an output row on its way out (padded: no bank conflicts)
constexpr uint32_t kF8StoreBytes = 32 * kF8RowBytes;  // a warp's 32 of them
constexpr uint32_t kF8TmemCols = 512;
constexpr int kF8Acc = 4, kF8AccCols = 128;  // accumulators
constexpr size_t kF8SmemBytes = 1024 + 1024 + static_cast<size_t>(kF8Stages) * kF8StageBytes +
                                kF8EpiWarps * kF8StoreBytes + kF8Ring * kF8Group * kF8Rows * sizeof(float2);

// Scales of x's rows (and of the hidden rows) are kept [block][row]: a k-block's are adjacent.
__host__ __device__ inline int64_t f8_row_pitch(int k) { return static_cast<int64_t>(fp8_blocks(k)) * kFp8Block; }

struct F8Args {
  int m, n, k;              // rows (Linear), weight rows per half, reduction length
  const float* sx;          // x's scales [blocks k][scale_rows]
  int64_t scale_rows;       // rows (positions) in all
  const float* ws;          // weight scales, contiguous [E][halves][blocks n][blocks k]
  const int4* groups;       // GateUp, Down (alut_fp8_grouped.cuh): (expert, first position, rows, 0)
  int group;                // Linear: tokens to a group, a multiple of 16
  const int* n_groups;
  const int* sorted;        // position -> slot
  int s;                    // slots per token
  uint8_t* hq;              // GateUp: [positions][f8_row_pitch(n)]
  float* hs;                // GateUp: [blocks n][scale_rows]
  void* out;                // Linear [m, n], Down [q, s, n]
  int out_dtype, out_vec;   // out_vec: 16-byte stores are aligned
  int64_t out_stride, out_stride_s;
  uint32_t* err;
  uint64_t wait_ns;         // how long a wait may take; 0: the call gives up before its first
};

// The same shared variable of the pair's CTA `rank`, as a shared::cluster address.
__device__ __forceinline__ uint32_t f8_of_rank(const void* p, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr(p)), "r"(rank));
  return r;
}
// No memory is handed over with this arrival (the accumulator was read, tcgen05 fences order that);
// with .release.cluster each one waited for the warp's memory traffic: 2 x the whole product's time.
__device__ __forceinline__ void f8_arrive_remote(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool f8_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool f8_test(uint32_t bar, uint32_t parity) {  // a look, without waiting
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
template <bool PAIR>
__device__ __forceinline__ void f8_give_up(volatile int* abort_flag) {
  *abort_flag = 1;
  if constexpr (PAIR) {
    uint32_t rank, there;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(smem_addr(const_cast<int*>(abort_flag))), "r"(rank ^ 1));
    asm volatile("st.shared::cluster.u32 [%0], 1;\n fence.acq_rel.cluster;" ::"r"(there) : "memory");
  }
}
// Waits of a whole warp on a barrier of this CTA (by its shared address); false: it ran out, or another
// role has given up (the flag and the error bit say so). The copies and each role's next tile stop then,
// and what is done until then stays in bounds. The timer is read only every 256 tries: a read of
// %globaltimer takes most of a microsecond.
// What must not happen is that warp 11 takes an accumulator for full that was filled out of turn, while
// the epilogue has yet to pass that barrier's last use (f8_drain says why).
//   One CTA: the lanes agree on the answer by a vote, and the MMA warp stops where one of its waits fails,
//   so no accumulator is filled out of turn before warp 11 itself has given up.
//   PAIR: the MMA warp serves two CTAs, and goes on for the rest of its tile (asking it there, or the vote,
//   took 2 % longer on 8192 x 4096 x 4096). A thread that gives up sets the flag of both CTAs first; what
//   follows out of turn comes after that, and warp 11 looks at its flag behind each wait.
template <bool PAIR>
__device__ __forceinline__ bool f8_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, const F8Args& a) {
  uint64_t t0 = 0;
  for (uint32_t n = 1; !(PAIR ? f8_try(bar, parity) : static_cast<bool>(__all_sync(0xffffffffu, f8_try(bar, parity)))); ++n) {
    if (n & 255) continue;
    bool over = *abort_flag;
    if (!over) {
      const uint64_t now = global_ns();
      if (t0 == 0) t0 = now;
      over = now - t0 > a.wait_ns;
      if (over && a.err) atomicOr(a.err, static_cast<uint32_t>(kErrMmaTimeout));
    }
    if (PAIR ? over : static_cast<bool>(__any_sync(0xffffffffu, over))) {
      f8_give_up<PAIR>(abort_flag);
      return false;
    }
  }
  return true;
}
// What warp 11 does once a call is given up: the epilogue's barriers from the `next`-th on (four per two
// k-blocks, in order), so that the epilogue comes to its end. A barrier is arrived at again only when the
// epilogue has passed its last use, which `passed` counts: a second arrival before that would complete a
// phase in place of an epilogue warp, whose bar.sync would then wait for good. (Until the call is given up
// the two keep step by themselves: an accumulator is full again only when the epilogue has released it.)
// The wait here comes without any copy or MMA; it is bounded by tries, not by the clock, which runs on while the GPU serves another process.
// (A loop of its own behind the other: as part of that one the product took 5 % longer.)
constexpr uint32_t kF8DrainTries = 1u << 24;
template <int ACC, int COUNT>
__device__ __forceinline__ void f8_drain(uint32_t passed, uint32_t next, uint32_t end) {
  for (; next < end; ++next) {
    const uint32_t ac = next % ACC, use = next / ACC;  // a fresh barrier counts as past parity 1
    for (uint32_t n = 0; n < kF8DrainTries && !f8_try(passed + 8 * ac, (use & 1) ^ 1); ++n) {
    }
    __syncwarp();
#pragma unroll
    for (int p = 0; p < 2; ++p) asm volatile("bar.arrive %0, %1;" ::"r"(1 + ACC * p + ac), "n"(COUNT) : "memory");
  }
}
// One lane of a converged warp, chosen so that the compiler knows it is one: the operands of the
// MMAs and copies then stay in uniform registers (behind lane == 0 the issue of a k-block's four
// MMAs and two commits took 600 cycles).
__device__ __forceinline__ bool f8_elect() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ void f8_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// TMA copy into this CTA's shared memory whose bytes count on a barrier of either CTA of the pair.
__device__ __forceinline__ void f8_load(void* dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
      "%3}], [%4];" ::"r"(smem_addr(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
// kind::f8f6f4 instruction descriptor: fp32 D, e4m3 A and B, K-major, M = 256, N = 128.
__host__ __device__ __forceinline__ uint32_t f8_idesc() {
  return (1u << 4) | (static_cast<uint32_t>(kF8AccCols >> 3) << 17) | (static_cast<uint32_t>(kF8PairRows >> 4) << 24);
}
// One accumulator of a k-block: 4 MMAs of K = 32 (descriptors advance by 32 bytes), then the commits
// that arrive in both CTAs: on `done`, and (LAST) on `freed`, the stage. A whole warp executes it and
// one elected lane issues; the election, the predicate and the operands (uniform registers) stay in
// one statement: as single instructions behind a branch the issue took 210 cycles a half k-block.
template <bool LAST>
__device__ __forceinline__ void f8_issue(uint32_t tmem, uint64_t dx, uint64_t dw, uint32_t idesc, uint32_t done,
                                         uint32_t freed) {
  if constexpr (LAST) {
    asm volatile(
        "{\n .reg .pred q, no, yes;\n .reg .b64 x, w;\n elect.sync _|q, 0xffffffff;\n"
        " setp.ne.b32 no, 0, 0;\n setp.eq.b32 yes, 0, 0;\n"
        " @q tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, no;\n"
        " add.u64 x, %1, 2;\n add.u64 w, %2, 2;\n"
        " @q tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], x, w, %3, yes;\n"
        " add.u64 x, %1, 4;\n add.u64 w, %2, 4;\n"
        " @q tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], x, w, %3, yes;\n"
        " add.u64 x, %1, 6;\n add.u64 w, %2, 6;\n"
        " @q tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], x, w, %3, yes;\n"
        " @q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%4], %6;\n"
        " @q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%5], %6;\n"
        "}\n" ::"r"(tmem),
        "l"(dx), "l"(dw), "r"(idesc), "r"(done), "r"(freed), "h"(static_cast<uint16_t>(3))
        : "memory");
  } else {
    asm volatile(
        "{\n .reg .pred q, no, yes;\n .reg .b64 x, w;\n elect.sync _|q, 0xffffffff;\n"
        " setp.ne.b32 no, 0, 0;\n setp.eq.b32 yes, 0, 0;\n"
        " @q tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, no;\n"
        " add.u64 x, %1, 2;\n add.u64 w, %2, 2;\n"
        " @q tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], x, w, %3, yes;\n"
        " add.u64 x, %1, 4;\n add.u64 w, %2, 4;\n"
        " @q tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], x, w, %3, yes;\n"
        " add.u64 x, %1, 6;\n add.u64 w, %2, 6;\n"
        " @q tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], x, w, %3, yes;\n"
        " @q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%4], %6;\n"
        "}\n" ::"r"(tmem),
        "l"(dx), "l"(dw), "r"(idesc), "r"(done), "r"(freed), "h"(static_cast<uint16_t>(3))
        : "memory");
  }
}

// 32 columns of this warp's 32 TMEM lanes, not waited for: the registers hold them after f8_ld_wait.
__device__ __forceinline__ void f8_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%"
      "19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
// Waits for this warp's loads; taking the registers in and out keeps every use behind it.
__device__ __forceinline__ void f8_ld_wait(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                 "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29])
               :
               : "memory");
  asm volatile("" : "+r"(r[30]), "+r"(r[31]));
}
// sum[j] += f * (the loaded column j). (The packed fma.rn.f32x2 is no help: it runs on one of the
// two fp32 pipes.)
__device__ __forceinline__ void f8_accumulate(float (&sum)[32], const uint32_t (&r)[32], float f) {
#pragma unroll
  for (int j = 0; j < 32; ++j) sum[j] = fmaf(__uint_as_float(r[j]), f, sum[j]);
}

// Output rows. A thread has 64 or 128 columns (from c0 on) of its row (offset o; negative: no row):
// into its own padded row of the warp's buffer, the offset behind it; then two rows at a time out.
template <typename TO, int C>
__device__ __forceinline__ void f8_store_row(TO* out, int64_t o, const float (&v)[C], int c0, int n, bool vec,
                                             unsigned char* rows) {
  static_assert(C * sizeof(TO) == 256, "a buffer row");
  constexpr int kPer = 16 / sizeof(TO);
  const int lane = threadIdx.x & 31;
  unsigned char* mine = rows + lane * kF8RowBytes;
  __syncwarp();
#pragma unroll
  for (int c = 0; c < C; c += kPer) {
    __align__(16) TO t[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) t[j] = from_f32<TO>(v[c + j]);
    *reinterpret_cast<uint4*>(mine + c * sizeof(TO)) = *reinterpret_cast<const uint4*>(t);
  }
  *reinterpret_cast<int64_t*>(mine + 256) = o;
  __syncwarp();
  const int have = min(C, n - c0);  // may be <= 0
  if (vec && have % kPer == 0) {
    const int c = (lane & 15) * kPer;
    const unsigned char* from = rows + (lane >> 4) * kF8RowBytes;
    TO* to = out + c0 + c;
    if (c < have) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int64_t ro = *reinterpret_cast<const int64_t*>(from + 2 * i * kF8RowBytes + 256);
        const uint4 u = *reinterpret_cast<const uint4*>(from + 2 * i * kF8RowBytes + (lane & 15) * 16);
        if (ro >= 0) *reinterpret_cast<uint4*>(to + ro) = u;
      }
    }
  } else {  // a ragged edge, or rows that do not start on 16 bytes: element by element along the rows
    for (int r = 0; r < 32; ++r) {
      const int64_t ro = *reinterpret_cast<const int64_t*>(rows + r * kF8RowBytes + 256);
      if (ro < 0) continue;
      for (int c = lane; c < have; c += 32)
        out[ro + c0 + c] = *reinterpret_cast<const TO*>(rows + r * kF8RowBytes + c * sizeof(TO));
    }
  }
}
// acc[i][h][j]: column c0 + 64 h + 32 i + j.
__device__ __forceinline__ void f8_store_rows(void* out, int64_t o, const float (&acc)[2][2][32], int c0, int n, int dtype,
                                              bool vec, unsigned char* rows) {
  float v[128];
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 32; ++j) v[64 * h + 32 * i + j] = acc[i][h][j];
  if (dtype == ALUT_BF16) {
    f8_store_row(static_cast<__nv_bfloat16*>(out), o, v, c0, n, vec, rows);
  } else if (dtype == ALUT_F16) {
    f8_store_row(static_cast<__half*>(out), o, v, c0, n, vec, rows);
  } else {
    f8_store_row(static_cast<float*>(out), o, reinterpret_cast<const float (&)[64]>(v[0]), c0, n, vec, rows);
    f8_store_row(static_cast<float*>(out), o, reinterpret_cast<const float (&)[64]>(v[64]), c0 + 64, n, vec, rows);
  }
}

__global__ void __launch_bounds__(kF8Threads, 1) __cluster_dims__(2, 1, 1)
    k_fp8_tc(const __grid_constant__ CUtensorMap x_map, const __grid_constant__ CUtensorMap w_map, F8Args a) {
  extern __shared__ unsigned char f8_raw[];
  unsigned char* f8_smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(f8_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(f8_smem);  // [kF8Stages] (the leader's counts for the pair)
  uint64_t* empty = full + kF8Stages;                  // [kF8Stages]
  uint64_t* t_full = empty + kF8Stages;                   // [kF8Acc]
  uint64_t* t_empty = t_full + kF8Acc;                    // [kF8Acc] (the leader's counts for the pair)
  uint64_t* f_full = t_empty + kF8Acc;                    // [kF8Ring]
  uint64_t* f_empty = f_full + kF8Ring;                   // [kF8Ring]
  uint64_t* passed = f_empty + kF8Ring;                   // [kF8Acc] (this CTA's epilogue)
  unsigned char* stages = f8_smem + 1024;                 // [kF8Stages][x rows | weight block]
  float2* ring = reinterpret_cast<float2*>(stages + kF8Stages * static_cast<size_t>(kF8StageBytes));  // [kF8Ring][kF8Group][kF8Rows]
  unsigned char* out_buf = reinterpret_cast<unsigned char*>(ring + kF8Ring * kF8Group * kF8Rows);    // output rows of 8 warps
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  volatile int* abort_flag = &s_abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = blockIdx.x & 1;  // in the pair
  const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;
  const int kblocks = fp8_blocks(a.k), nblocks = fp8_blocks(a.n);
  if (warp == kF8MmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&s_tmem)),
                 "r"(kF8TmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  if (tid == 0) {
    for (int i = 0; i < kF8Stages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < kF8Acc; ++i) {
      mbar_init(&t_full[i], 1);
      mbar_init(&t_empty[i], 2 * kF8EpiWarps);
      mbar_init(&passed[i], kF8EpiWarps);
    }
    for (int i = 0; i < kF8Ring; ++i) {
      mbar_init(&f_full[i], 1);
      mbar_init(&f_empty[i], kF8EpiWarps);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    s_abort = a.wait_ns == 0;
    if (a.wait_ns == 0 && a.err) atomicOr(a.err, static_cast<uint32_t>(kErrMmaTimeout));
  }
  tc_fence_before();
  __syncthreads();
  f8_cluster_sync();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  pdl_wait();  // x's 8-bit rows and scales come from the kernel before; no later kernel is let ahead
  const int nt = (nblocks + 1) / 2, mt = (a.m + kF8PairRows - 1) / kF8PairRows;
  const int ntiles = mt * nt;  // (the host refuses more than fit)
  const int step_m = npairs / nt, step_n = npairs % nt;
  // The tiles of this pair, without a division per tile: row tile mi, column tile ni.
  struct Tile {
    int i, mi, ni;
  };
  auto first_tile = [&]() { return Tile{pair, pair / nt, pair % nt}; };
  auto next_tile = [&](Tile t) {
    t.i += npairs;
    t.mi += step_m;
    t.ni += step_n;
    if (t.ni >= nt) {
      t.ni -= nt;
      ++t.mi;
    }
    return t;
  };
  auto wait = [&](uint64_t* bars, int i, uint32_t parity) {  // a fresh barrier counts as past parity 1
    return f8_wait<true>(smem_addr(bars) + 8 * i, parity, abort_flag, a);
  };
  auto stopped = [&]() { return __any_sync(0xffffffffu, *abort_flag); };

  // Every role is a whole warp that walks the same tiles; one elected lane issues.
  if (warp >= kF8EpiWarps) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kF8RoleRegs));
    if (warp == kF8CopyWarp) {
      // ---- TMA copies --------------------------------------------------------------------------
      int st = 0, past = 1;
      for (Tile t = first_tile(); t.i < ntiles && !stopped(); t = next_tile(t)) {
        const bool second = a.m - t.mi * kF8PairRows > kF8Rows;  // the second CTA has rows
        const uint32_t bytes = kF8TileBytes * (second ? 4 : 3);
        const int wrow = (2 * t.ni + static_cast<int>(rank)) * kFp8Block;
        const int xrow = t.mi * kF8PairRows + static_cast<int>(rank) * kF8Rows;
        for (int kb = 0; kb < kblocks; ++kb, (++st == kF8Stages ? (st = 0, past ^= 1) : 0)) {
          const bool free = wait(empty, st, past);
          if (f8_elect() && free) {
            unsigned char* sx = stages + static_cast<size_t>(st) * kF8StageBytes;
            const uint32_t bar = f8_of_rank(&full[st], 0);
            if (rank == 0) mbar_expect_tx(&full[st], bytes);
            f8_load(sx + kF8TileBytes, &w_map, kb * kFp8Block, wrow, bar);
            if (rank == 0 || second) f8_load(sx, &x_map, kb * kFp8Block, xrow, bar);
          }
          __syncwarp();
        }
      }
    } else if (warp == kF8MmaWarp) {
      // ---- MMA issuer ----------------------------------------------------------------------------
      if (rank == 0) {
        int st = 0, ph = 0, buf = 0, past = 1;
        const uint32_t done0 = smem_addr(t_full), freed0 = smem_addr(empty), full0 = smem_addr(full), empty0 = smem_addr(t_empty);
        bool seen_full = false, seen0 = false, seen1 = false;
        const uint32_t idesc = f8_idesc();
        const uint64_t desc0 = pt_desc_sw128(smem_addr(stages));  // + address / 16 within the first 14 bits
        for (int tile = pair; tile < ntiles && !stopped(); tile += npairs) {
          for (int kb = 0; kb < kblocks; ++kb) {
            // accumulators 2 buf and 2 buf + 1, each used once per two k-blocks
            const uint64_t dx = desc0 + static_cast<uint32_t>(st) * (kF8StageBytes >> 4), dw = dx + (kF8TileBytes >> 4);
            const uint32_t d = tmem + 2 * buf * kF8AccCols, done = done0 + 16 * buf, freed = freed0 + 8 * st;
            if (!seen_full) wait(full, st, ph);
            if (!seen0) wait(t_empty, 2 * buf, past);
            tc_fence_after();
            f8_issue<false>(d, dx, dw, idesc, done, 0);
            if (!seen1) wait(t_empty, 2 * buf + 1, past);
            tc_fence_after();
            if (++st == kF8Stages) {
              st = 0;
              ph ^= 1;
            }
            past ^= buf;
            buf ^= 1;
            // A look at the next k-block's barriers: the answers arrive behind this issue. (A wait
            // costs 100 cycles and more even where it is over, three of them more than the MMAs.)
            seen_full = f8_test(full0 + 8 * st, ph);
            seen0 = f8_test(empty0 + 16 * buf, past);
            seen1 = f8_test(empty0 + 16 * buf + 8, past);
            f8_issue<true>(d + kF8AccCols, dx, dw + (kF8TileBytes >> 5), idesc, done + 8, freed);
          }
        }
      }
    } else if (warp == kF8ScaleWarp) {
      // ---- factors -----------------------------------------------------------------------------
      // A ring slot's 24 values are loaded together, and the next slot's before this one's are
      // written: loads one k-block at a time made this warp the bottleneck (their L2 latency, 860
      // cycles a k-block).
      int sl = 0, past = 1;
      for (Tile t = first_tile(); t.i < ntiles && !stopped(); t = next_tile(t)) {
        const int row0 = t.mi * kF8PairRows + static_cast<int>(rank) * kF8Rows;
        const int rows = min(kF8Rows, a.m - row0);  // may be <= 0
        const float* sx = a.sx + row0 + lane;
        const float* sw0 = a.ws + static_cast<int64_t>(2 * t.ni) * kblocks;
        const float* sw1 = 2 * t.ni + 1 < nblocks ? sw0 + kblocks : sw0;  // (none past the last)
        float s[kF8Group][4], w[kF8Group][2];
        auto load = [&](int kb0) {
#pragma unroll
          for (int i = 0; i < kF8Group; ++i) {
            const bool on = kb0 + i < kblocks;
            const float* p = sx + (kb0 + i) * a.scale_rows;
#pragma unroll
            for (int j = 0; j < 4; ++j) s[i][j] = on && lane + 32 * j < rows ? __ldcg(p + 32 * j) : 0.f;
            w[i][0] = on ? __ldg(sw0 + kb0 + i) : 0.f;
            w[i][1] = on ? __ldg(sw1 + kb0 + i) : 0.f;
          }
        };
        load(0);
        for (int kb0 = 0; kb0 < kblocks; kb0 += kF8Group) {
          wait(f_empty, sl, past);
#pragma unroll
          for (int i = 0; i < kF8Group; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              ring[(sl * kF8Group + i) * kF8Rows + lane + 32 * j] = make_float2(s[i][j] * w[i][0], s[i][j] * w[i][1]);
          if (kb0 + kF8Group < kblocks) load(kb0 + kF8Group);
          __syncwarp();
          if (lane == 0) mbar_arrive(&f_full[sl]);
          if (++sl == kF8Ring) {
            sl = 0;
            past ^= 1;
          }
        }
      }
    } else {
      // ---- accumulators (and their factors) done: let the epilogue go ------------------------------
      // The factors of k-block kb + 1 are there when the epilogue passes the barrier of (kb, 1).
      int sl = 0, sph = 0, buf = 0, ph = 0;
      auto factors = [&](int kb) {
        if (kb & (kF8Group - 1)) return;
        wait(f_full, sl, sph);
        if (++sl == kF8Ring) {
          sl = 0;
          sph ^= 1;
        }
      };
      uint32_t gone = 0;  // k-blocks of the tiles before this one
      bool given_up = a.wait_ns == 0;
      int kb = 0, h = 0;
      for (int tile = pair; tile < ntiles && !given_up; tile += npairs) {
        factors(0);
        for (kb = 0; kb < kblocks; ++kb) {
#pragma unroll
          for (h = 0; h < 2; ++h) {
            if (h == 1 && kb + 1 < kblocks) factors(kb + 1);
            wait(t_full, 2 * buf + h, ph);
            given_up = stopped();
            if (given_up) break;
#pragma unroll
            for (int p = 0; p < 2; ++p)
              asm volatile("bar.arrive %0, %1;" ::"r"(1 + kF8Acc * p + 2 * buf + h), "n"(32 * (kF8EpiWarps / 2 + 1)) : "memory");
          }
          if (given_up) break;
          ph ^= buf;
          buf ^= 1;
        }
        if (!given_up) gone += kblocks;
      }
      if (given_up) {
        f8_give_up<true>(abort_flag);
        const uint32_t tiles = pair < ntiles ? (ntiles - pair + npairs - 1) / npairs : 0;
        f8_drain<kF8Acc, 32 * (kF8EpiWarps / 2 + 1)>(smem_addr(passed), a.wait_ns == 0 ? 0 : 2 * (gone + kb) + h,
                                                     2 * tiles * kblocks);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kF8EpiRegs));
    // ---- epilogue ------------------------------------------------------------------------------
    const int part = warp >> 2;
    const int warp_row = (warp & 3) * 32, row = warp_row + lane;
    const uint32_t lane_base = tmem + (static_cast<uint32_t>(warp_row) << 16);
    const int col0 = part * 64, col1 = col0 + 32;
    const uint32_t released = lane == 0 ? f8_of_rank(&t_empty[0], 0) : f8_of_rank(&passed[0], rank);
    unsigned char* buf_out = out_buf + warp * kF8StoreBytes;
    int buf = 0, sl = 0;
    // The two column parts go by barriers of their own: warps w and w + 4 share a scheduler, and one
    // adds while the other waits for its load.
    auto ready = [&](int ac) {
      asm volatile("bar.sync %0, %1;" ::"r"(1 + kF8Acc * part + ac), "n"(32 * (kF8EpiWarps / 2 + 1)) : "memory");
      tc_fence_after();
    };
    auto release = [&](int ac) {
      tc_fence_before();
      __syncwarp();
      if (lane < 2) f8_arrive_remote(released + 8 * ac);
    };
    auto group_read = [&](int kb) {  // this warp has the factors of k-block kb: its group's last?
      if ((kb & (kF8Group - 1)) == kF8Group - 1 || kb == kblocks - 1) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&f_empty[sl]);
        if (++sl == kF8Ring) sl = 0;
      }
    };
    for (Tile t = first_tile(); t.i < ntiles; t = next_tile(t)) {
      const int row0 = t.mi * kF8PairRows + static_cast<int>(rank) * kF8Rows;
      const int rows = a.m - row0;  // of this CTA; may be <= 0
      const bool warp_live = warp_row < rows;
      // where this thread's row of outputs begins
      const int64_t o = row < rows ? static_cast<int64_t>(row0 + row) * a.out_stride : -1;
      float acc[2][2][32];  // [col0, col1][half of the k-block's accumulators][column]
#pragma unroll
      for (int j = 0; j < 32; ++j) acc[0][0][j] = acc[0][1][j] = acc[1][0][j] = acc[1][1][j] = 0.f;
      if (warp_live) {
        // A load is under way while the registers of the one before are added up: the next
        // accumulator's first 32 columns behind this one's, the last 32 behind those.
        uint32_t v0[32], v1[32];
        const float2* fr = ring + row;
        float f, fn = 0.f;
        ready(2 * buf);
        auto factors = [&](int kb) {
          const float2 both = fr[(sl * kF8Group + (kb & (kF8Group - 1))) * kF8Rows];
          group_read(kb);
          return part ? both.y : both.x;  // one weight block
        };
        f = factors(0);
        f8_ld32(lane_base + 2 * buf * kF8AccCols + col0, v0);
        f8_ld32(lane_base + 2 * buf * kF8AccCols + col1, v1);
        for (int kb = 0; kb < kblocks; ++kb) {
          const uint32_t d = lane_base + 2 * buf * kF8AccCols, dn = lane_base + 2 * (buf ^ 1) * kF8AccCols;
          f8_ld_wait(v0);
          f8_ld_wait(v1);
          release(2 * buf);
          f8_accumulate(acc[0][0], v0, f);
          ready(2 * buf + 1);
          f8_ld32(d + kF8AccCols + col0, v0);
          const bool more = kb + 1 < kblocks;
          if (more) fn = factors(kb + 1);
          f8_accumulate(acc[1][0], v1, f);
          f8_ld32(d + kF8AccCols + col1, v1);
          f8_ld_wait(v0);
          f8_ld_wait(v1);
          release(2 * buf + 1);
          f8_accumulate(acc[0][1], v0, f);
          if (more) {
            ready(2 * (buf ^ 1));
            f8_ld32(dn + col0, v0);
          }
          f8_accumulate(acc[1][1], v1, f);
          if (more) f8_ld32(dn + col1, v1);
          f = fn;
          buf ^= 1;
        }
      } else {  // no row here: nothing to read
        for (int kb = 0; kb < kblocks; ++kb, buf ^= 1) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            ready(2 * buf + h);
            release(2 * buf + h);
          }
          group_read(kb);
        }
      }
      if (warp_live) f8_store_rows(a.out, o, acc, (2 * t.ni + part) * kFp8Block, a.n, a.out_dtype, a.out_vec, buf_out);
    }
  }

  __syncthreads();
  if (*abort_flag && tid == 0) {  // what is in flight gets 10 ms to end before the memory goes
    const uint64_t t0 = global_ns();
    while (global_ns() - t0 < 10000000ull) __nanosleep(1000);
  }
  tc_fence_before();
  __syncthreads();
  f8_cluster_sync();  // neither CTA leaves while the other still uses its memory
  if (warp == kF8MmaWarp)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kF8TmemCols) : "memory");
}

// ---- what the products need first ------------------------------------------------------------

struct F8PrepArgs {
  const void* x;
  int64_t x_stride;
  int rows, k, x_vec;
  uint8_t* xq;  // [rows or positions][f8_row_pitch(k)], columns from k on zero
  float* sx;    // [blocks][scale_rows]
  int64_t scale_rows;
  const int* place;  // [rows][s] position of each slot, -1: not computed; NULL: a row is its own position
  int s;
  void* out;         // with place: rows of slots that are not computed are set to 0 (NULL: left alone)
  int out_dtype, out_vec;
  int64_t out_stride, out_stride_s;
};

// x's 8-bit form. Memory-bound: 8192 x 4096 bf16 23 us (4.4 TB/s), 4096 x 2048 into 19700 places with
// 13100 rows of zeros 22 us (5.1 TB/s). A warp takes kF8RowBlocks blocks of a row at a time, two side by side (16 lanes of 8
// columns each); the next unit's loads are under way while this one is converted and stored. With
// `place` the first unit overlaps the plan up to its stores.
constexpr int kF8RowBlocks = 8;
constexpr int kF8RowCtas = 4;  // per SM: 32 warps with 2 KB each on the way
template <typename TX>
__global__ void __launch_bounds__(256, kF8RowCtas) k_fp8_rows(F8PrepArgs a) {
  constexpr int kU = kF8RowBlocks / 2;
  pdl_launch_dependents();
  const int kb = fp8_blocks(a.k), chunks = (kb + kF8RowBlocks - 1) / kF8RowBlocks;
  const int units = a.rows * chunks;  // (the host keeps them below 2^31)
  const int step = gridDim.x * 8, step_r = step / chunks, step_c = step - step_r * chunks;
  int unit = blockIdx.x * 8 + (threadIdx.x >> 5);
  int row = unit / chunks, chunk = unit - row * chunks;
  const int lane = threadIdx.x & 31, sub = lane & 15, side = lane >> 4;
  auto fetch = [&](F8Raw8<TX> (&r)[kU], int row, int chunk) {
    const TX* src = static_cast<const TX*>(a.x) + row * a.x_stride;
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int c = (chunk * kF8RowBlocks + side + 2 * u) * kFp8Block + sub * 8;
      if (a.x_vec && c + 8 <= a.k) {
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(TX) / 2); ++i) r[u].w[i] = __ldg(reinterpret_cast<const uint4*>(src + c) + i);
      } else {
        TX* e = reinterpret_cast<TX*>(&r[u]);
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = c + j < a.k ? src[c + j] : from_f32<TX>(0.f);
      }
    }
  };
  F8Raw8<TX> raw[kU];
  if (unit < units) fetch(raw, row, chunk);
  bool planned = !a.place;
  while (unit < units) {
    const int r = row, b0 = chunk * kF8RowBlocks + side;
    uint2 q[kU];
    float s[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      float v[8];
      f8_widen<TX>(raw[u], v);
      uint32_t m = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) m = max(m, abs_bits(v[j]));
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
      const float am = fp8_amax(m);
      const float f = kE4m3Max / am;
      s[u] = am / kE4m3Max;
      q[u].x = e4m3x4(v[0] * f, v[1] * f, v[2] * f, v[3] * f);
      q[u].y = e4m3x4(v[4] * f, v[5] * f, v[6] * f, v[7] * f);
    }
    unit += step;
    row += step_r;
    chunk += step_c;
    if (chunk >= chunks) {
      chunk -= chunks;
      ++row;
    }
    if (unit < units) fetch(raw, row, chunk);
    auto put = [&](int64_t p) {
      uint8_t* dst = a.xq + p * f8_row_pitch(a.k) + sub * 8;
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const int b = b0 + 2 * u;
        if (b >= kb) break;
        *reinterpret_cast<uint2*>(dst + b * kFp8Block) = q[u];
        if (sub == 0) a.sx[b * a.scale_rows + p] = s[u];
      }
    };
    if (!a.place) {
      put(r);
      continue;
    }
    if (!planned) pdl_wait();  // the plan
    planned = true;
    int places = -1;  // of 32 slots, a lane each: one load's latency for all
    for (int t = 0; t < a.s; ++t) {
      if ((t & 31) == 0 && t + lane < a.s) places = __ldcg(a.place + static_cast<int64_t>(r) * a.s + t + lane);
      const int p = __shfl_sync(0xffffffffu, places, t & 31);
      if (p >= 0) {
        put(p);
      } else if (a.out) {
        const int64_t o = r * a.out_stride + t * a.out_stride_s;
#pragma unroll
        for (int u = 0; u < kU; ++u) {
          const int c = (b0 + 2 * u) * kFp8Block + sub * 8;
          if (a.out_vec && c + 8 <= a.k) {
            const float z[8] = {};
            if (a.out_dtype == ALUT_BF16) store8(static_cast<__nv_bfloat16*>(a.out) + o + c, z);
            else if (a.out_dtype == ALUT_F16) store8(static_cast<__half*>(a.out) + o + c, z);
            else store8(static_cast<float*>(a.out) + o + c, z);
          } else {
            for (int j = 0; j < 8; ++j)
              if (c + j < a.k) store_any(a.out, o + c + j, 0.f, a.out_dtype);
          }
        }
      }
    }
  }
}

// The plan: computed slots grouped by expert, by one cluster of CTAs that share the slots. Each
// counts its share per expert in shared memory; after a cluster barrier every CTA knows the counts
// before its own (distributed shared memory) and places its slots, in any order within an expert (a
// row's result does not depend on its place). groups[i] = (expert, first position, rows <=
// group_rows (a multiple of 16), 0), an expert's as equal as steps of 16 allow. 32768 slots
// take 11 us, one CTA took 42; 128 slots 6.4 either way (two launches' worth of latency).
constexpr int kF8PlanThreads = 1024;
constexpr int kF8PlanCtas = 8;

__global__ void __launch_bounds__(kF8PlanThreads) __cluster_dims__(kF8PlanCtas, 1, 1)
    k_fp8_plan(Fp8Route r, int group_rows, int* sorted, int* place, int4* groups, int* n_groups) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  extern __shared__ int plan_smem[];
  int* count = plan_smem;       // [E] this CTA's slots per expert
  int* next = plan_smem + r.e;  // [E] next position
  __shared__ int s_warp[32][2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = static_cast<int>(cluster.block_rank());
  const int n = r.q * r.s;
  const int step = kF8PlanThreads * kF8PlanCtas;
  pdl_launch_dependents();
  for (int e = tid; e < r.e; e += kF8PlanThreads) count[e] = 0;
  __syncthreads();
  bool bad = false;
#pragma unroll 4
  for (int64_t i = rank * kF8PlanThreads + tid; i < n; i += step) {
    const int e = fp8_slot_expert(r, static_cast<int>(i), bad);
    if (e >= 0) atomicAdd(&count[e], 1);
  }
  if (bad && r.err) atomicOr(r.err, static_cast<uint32_t>(kErrBadExpert));
  cluster.sync();
  // Exclusive prefix of (slots, groups) over the experts, two consecutive experts per thread.
  int c[2], g[2], per[2], mine[2];  // mine: slots of the CTAs before this one
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int e = 2 * tid + j;
    c[j] = mine[j] = 0;
    if (e < r.e) {
#pragma unroll
      for (int k = 0; k < kF8PlanCtas; ++k) {
        const int v = cluster.map_shared_rank(count, k)[e];
        c[j] += v;
        if (k < rank) mine[j] += v;
      }
    }
    g[j] = (c[j] + group_rows - 1) / group_rows;
    per[j] = g[j] ? ((c[j] + g[j] - 1) / g[j] + 15) / 16 * 16 : 0;  // equal groups, in steps of 16 rows
  }
  int sc = c[0] + c[1], sg = g[0] + g[1];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int pc = __shfl_up_sync(0xffffffffu, sc, o), pg = __shfl_up_sync(0xffffffffu, sg, o);
    if (lane >= o) {
      sc += pc;
      sg += pg;
    }
  }
  if (lane == 31) {
    s_warp[warp][0] = sc;
    s_warp[warp][1] = sg;
  }
  __syncthreads();
  int bc = 0, bg = 0;
  for (int w = 0; w < warp; ++w) {
    bc += s_warp[w][0];
    bg += s_warp[w][1];
  }
  int pos = bc + sc - c[0] - c[1], gi = bg + sg - g[0] - g[1];
  if (rank == 0 && tid == kF8PlanThreads - 1) *n_groups = bg + sg;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int e = 2 * tid + j;
    if (e < r.e) {
      next[e] = pos + mine[j];
      if (rank == 0)
        for (int k = 0; k < g[j]; ++k)
          groups[gi + k] = make_int4(e, pos + k * per[j], min(per[j], c[j] - k * per[j]), 0);
    }
    pos += c[j];
    gi += g[j];
  }
  __syncthreads();
#pragma unroll 4
  for (int64_t i = rank * kF8PlanThreads + tid; i < n; i += step) {
    const int e = fp8_slot_expert(r, static_cast<int>(i), bad);
    int p = -1;
    if (e >= 0) {
      p = atomicAdd(&next[e], 1);
      sorted[p] = static_cast<int>(i);
    }
    place[i] = p;
  }
  cluster.sync();  // no CTA leaves while another reads its counts
}

}  // namespace alut
