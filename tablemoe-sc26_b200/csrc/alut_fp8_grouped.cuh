// Block-scaled e4m3 products for tokens in groups: tcgen05 (kind::f8f6f4) with the weights as the M
// operand and a group of tokens as N. The routed experts of more than 8 slots, and the plain product of
// up to some hundred rows (one tile per SM: linear_group).
//
// An expert gets any number of tokens: 25 of a short prompt, 154 of a long one. With tokens as M (256
// to a pair of CTAs) a tile costs 256 of them whether they are there or not; as N a group takes what it
// has, in steps of 16 up to 128 (the plan cuts an expert's tokens into groups as equal as that allows).
// A tile is two 128-row weight blocks x one group: the gate and the up rows of 128 hidden units
// (GateUp), or 256 adjacent outputs (Down, Linear). Per 128 columns of K a CTA copies 32 KB of weights
// and 128 bytes a token. x's rows lie in the order of the plan (k_fp8_rows writes a token's 8-bit row once per
// computed slot): gathering them here was slower (tile::gather4 moves a 128-byte row every 13 ns).
// As in alut_fp8_tc.cuh an accumulator holds one k-block of one weight block (the scales change with
// each): four of 128 columns in tensor memory, each added up, times sx[token, block] sw[block], in fp32
// registers.
//
//   warps 0-7  epilogue: TMEM lane quarter warp % 4, first or second half of the group's tokens
//   warp 8     TMA copies (128-byte swizzle; the tokens' rows 16 at a time)
//   warp 9     MMA issuer
//   warp 10    the scales of a k-block, into a ring in shared memory
//   warp 11    waits for accumulators and scales and lets the epilogue go by named barriers
// TMEM is read 16 lanes x 8 columns at a time (16x256b): a thread has 4 weight rows of 2 tokens in each
// 8, so that it needs a quarter of the group's scales. With a lane per row (32x32b) every sum needed
// its own, and reading them (16 bytes per lane and 4 tokens) took longer than anything else: 182 + 146
// us (GateUp + Down of the first case below), 146 + 112 with this layout. The same fragments go out
// transposed by stmatrix, 32 to 64 adjacent bytes of a token at a time. Sums, scales and silu are taken
// two tokens at a time (f32x2): that, and a tile's end in less code, brought it to 136 + 93; a quarter
// of the epilogue's time was the wait for instructions, of which each is used once per tile.
// GateUp ends with h = silu(gate) up in its 8-bit form: the 128 rows of the tile are one block of the
// next product, whose maximum per token is a reduction over 8 lanes and over the four quarters.
//
// Measured, 4096 tokens x 8 slots (60 % computed) over 128 experts of 2048 x 768: GateUp 136, Down 93
// us (with 256 tokens to a tile of a pair of CTAs 160 and 105); 300 x 6 over 72 experts of 2560 x 1280:
// 78 and 50 us (130 and 75), 6.1 and 4.7 TB/s of weights, with groups of up to 48 tokens (of up to 128:
// 88 and 53); 16 x 8 over the 128 experts 36 and 20 us, 4.5 TB/s. Copies and MMAs alone take 124 us of
// the first pair: 710 cycles a k-block for 80 tokens. In the first case the epilogue bounds it (1050
// cycles a k-block, and some 4000 of a tile's end during which the MMAs run two k-blocks ahead at
// most); sixteen epilogue warps instead of eight, with half the sums each, took 173 + 139. In the
// others memory does.
// Waits are bounded, and an abort ends, as in alut_fp8_tc.cuh.
#pragma once

#include <type_traits>

#include "alut_fp8_tc.cuh"

namespace alut {

constexpr int kG8Tokens = 128;  // per group
constexpr int kG8Step = 16;     // a group's tokens are copied and multiplied in steps of
constexpr int kG8Stages = 4;
constexpr int kG8OutBytes = 16 * 48;  // per warp, twice: outputs on their way out
constexpr uint32_t kG8StageBytes = 3 * kF8TileBytes;  // two weight blocks, the tokens' rows
constexpr size_t kG8SmemBytes = 1024 + 1024 + static_cast<size_t>(kG8Stages) * kG8StageBytes +
                                kF8Ring * kF8Group * (kG8Tokens * sizeof(float) + sizeof(float2));

__device__ __forceinline__ void g8_load_weight(void* dst, const CUtensorMap* map, int x, int y, int half, int e,
                                               uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(smem_addr(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(half), "r"(e), "r"(smem_addr(bar))
      : "memory");
}
// One accumulator: 4 MMAs of K = 32, then the commit on `done` and (LAST) on `freed`; see f8_issue.
template <bool LAST>
__device__ __forceinline__ void g8_issue(uint32_t tmem, uint64_t dw, uint64_t dx, uint32_t idesc, uint32_t done,
                                         uint32_t freed) {
  if constexpr (LAST) {
    asm volatile(
        "{\n .reg .pred q, no, yes;\n .reg .b64 x, w;\n elect.sync _|q, 0xffffffff;\n"
        " setp.ne.b32 no, 0, 0;\n setp.eq.b32 yes, 0, 0;\n"
        " @q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, no;\n"
        " add.u64 w, %1, 2;\n add.u64 x, %2, 2;\n"
        " @q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], w, x, %3, yes;\n"
        " add.u64 w, %1, 4;\n add.u64 x, %2, 4;\n"
        " @q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], w, x, %3, yes;\n"
        " add.u64 w, %1, 6;\n add.u64 x, %2, 6;\n"
        " @q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], w, x, %3, yes;\n"
        " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%4];\n"
        " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%5];\n"
        "}\n" ::"r"(tmem),
        "l"(dw), "l"(dx), "r"(idesc), "r"(done), "r"(freed)
        : "memory");
  } else {
    asm volatile(
        "{\n .reg .pred q, no, yes;\n .reg .b64 x, w;\n elect.sync _|q, 0xffffffff;\n"
        " setp.ne.b32 no, 0, 0;\n setp.eq.b32 yes, 0, 0;\n"
        " @q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, no;\n"
        " add.u64 w, %1, 2;\n add.u64 x, %2, 2;\n"
        " @q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], w, x, %3, yes;\n"
        " add.u64 w, %1, 4;\n add.u64 x, %2, 4;\n"
        " @q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], w, x, %3, yes;\n"
        " add.u64 w, %1, 6;\n add.u64 x, %2, 6;\n"
        " @q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], w, x, %3, yes;\n"
        " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%4];\n"
        "}\n" ::"r"(tmem),
        "l"(dw), "l"(dx), "r"(idesc), "r"(done), "r"(freed)
        : "memory");
  }
}
// 16 lanes x 8 C columns of TMEM, not waited for (g8_ld_wait). Lane l of the warp gets rows l / 4 and
// l / 4 + 8 of columns 2 (l % 4) and the next of each 8: r[column / 8][2 row + column].
template <int C, int O = 0>
__device__ __forceinline__ void g8_ld(uint32_t t, float (&r)[C][4]) {
  if constexpr (C - O >= 4) {
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=f"(r[O][0]), "=f"(r[O][1]), "=f"(r[O][2]), "=f"(r[O][3]), "=f"(r[O + 1][0]), "=f"(r[O + 1][1]),
                   "=f"(r[O + 1][2]), "=f"(r[O + 1][3]), "=f"(r[O + 2][0]), "=f"(r[O + 2][1]), "=f"(r[O + 2][2]),
                   "=f"(r[O + 2][3]), "=f"(r[O + 3][0]), "=f"(r[O + 3][1]), "=f"(r[O + 3][2]), "=f"(r[O + 3][3])
                 : "r"(t + 8 * O)
                 : "memory");
    if constexpr (C > O + 4) g8_ld<C, O + 4>(t, r);
  } else if constexpr (C - O >= 2) {
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=f"(r[O][0]), "=f"(r[O][1]), "=f"(r[O][2]), "=f"(r[O][3]), "=f"(r[O + 1][0]), "=f"(r[O + 1][1]),
                   "=f"(r[O + 1][2]), "=f"(r[O + 1][3])
                 : "r"(t + 8 * O)
                 : "memory");
    if constexpr (C > O + 2) g8_ld<C, O + 2>(t, r);
  } else {
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x1.b32 {%0,%1,%2,%3}, [%4];"
                 : "=f"(r[O][0]), "=f"(r[O][1]), "=f"(r[O][2]), "=f"(r[O][3])
                 : "r"(t + 8 * O)
                 : "memory");
  }
}
// What is loaded is there: no use of r moves above this.
template <int C>
__device__ __forceinline__ void g8_ld_wait(float (&r)[C][4]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < C; ++i) asm volatile("" : "+f"(r[i][0]), "+f"(r[i][1]), "+f"(r[i][2]), "+f"(r[i][3]));
}
// Two fp32 numbers in one register pair: the FMA units take both with one instruction.
__device__ __forceinline__ uint64_t g8_pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 g8_unpair(uint64_t p) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p));
  return r;
}
__device__ __forceinline__ uint64_t g8_mul(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t g8_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t g8_add(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// silu_mul of both.
__device__ __forceinline__ uint64_t g8_silu_mul(uint64_t g, uint64_t u) {
  const float2 t = g8_unpair(g8_mul(g, g8_pair(-kLog2E, -kLog2E)));
  const float2 e = g8_unpair(g8_add(g8_pair(exp2_approx(t.x), exp2_approx(t.y)), g8_pair(1.0f, 1.0f)));
  return g8_mul(g8_mul(g, g8_pair(rcp_approx(e.x), rcp_approx(e.y))), u);
}
// The larger of m >= 0 and |x|; a NaN wins.
__device__ __forceinline__ float g8_max_abs(float m, float x) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(m), "f"(fabsf(x)));
  return r;
}
// Four (two) 8 x 8 matrices of 16-bit elements in that layout, stored transposed: lane 8 m + j gives the
// address of the 16 bytes of matrix m's column j.
__device__ __forceinline__ void g8_store_matrices(unsigned char* p, uint32_t m0, uint32_t m1, uint32_t m2, uint32_t m3) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(smem_addr(p)), "r"(m0),
               "r"(m1), "r"(m2), "r"(m3)
               : "memory");
}
__device__ __forceinline__ void g8_store_matrices(unsigned char* p, uint32_t m0, uint32_t m1) {
  asm volatile("stmatrix.sync.aligned.m8n8.x2.trans.shared.b16 [%0], {%1, %2};" ::"r"(smem_addr(p)), "r"(m0), "r"(m1)
               : "memory");
}
template <typename TO>
__device__ __forceinline__ uint32_t g8_pack(float lo, float hi) {
  if constexpr (std::is_same_v<TO, __half>) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}
// A Down tile's outputs of one weight block: TMEM's rows are output columns (`n` left from `out` on),
// its columns tokens, `tokens` of them there, whose outputs begin at off[]. acc[16-row half][8 tokens][..].
// VEC: all 32 outputs are there, on 16 bytes. (The two cases are two loops, each short straight code: a
// tile's end is bound by the instructions' way into the SM.)
template <typename TO, bool VEC, int C>
__device__ __forceinline__ void g8_store(TO* out, int n, const float (&acc)[2][C][4], const int64_t* off,
                                         unsigned char (*stage)[kG8OutBytes], int tokens, int lane) {
  if constexpr (sizeof(TO) == 4) {
#pragma unroll
    for (int i = 0; i < C * 8; ++i) {
      const int h = i / (4 * C), c = i / 4 % C, t = 8 * c + 2 * (lane & 3) + (i & 1), row = 16 * h + 8 * (i >> 1 & 1) + lane / 4;
      if (t < tokens && row < n) out[off[t] + row] = from_f32<TO>(acc[h][c][i & 3]);
    }
  } else {
    // through shared memory: rows of 32 outputs (64 bytes, 16 more against bank conflicts)
    constexpr int kVec = 8;
    __syncwarp();
    const int col = (lane & 3) * kVec;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      unsigned char* buf = stage[c & 1];
      g8_store_matrices(buf + (lane & 7) * 80 + (lane >> 3) * 16, g8_pack<TO>(acc[0][c][0], acc[0][c][1]),
                        g8_pack<TO>(acc[0][c][2], acc[0][c][3]), g8_pack<TO>(acc[1][c][0], acc[1][c][1]),
                        g8_pack<TO>(acc[1][c][2], acc[1][c][3]));
      __syncwarp();
      const int t = 8 * c + lane / 4;
      const uint4 u = *reinterpret_cast<const uint4*>(buf + (lane / 4) * 80 + (lane & 3) * 16);
      if (t < tokens) {
        TO* p = out + off[t] + col;
        if constexpr (VEC) {
          *reinterpret_cast<uint4*>(p) = u;
        } else {
          const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
          for (int j = 0; j < kVec; ++j)
            if (col + j < n) reinterpret_cast<uint16_t*>(p)[j] = static_cast<uint16_t>(w[j >> 1] >> (j & 1) * 16);
        }
      }
    }
  }
}

template <int MODE>
__global__ void __launch_bounds__(kF8Threads, 1)
    k_fp8_grouped(const __grid_constant__ CUtensorMap x_map, const __grid_constant__ CUtensorMap w_map, F8Args a) {
  extern __shared__ unsigned char g8_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(g8_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem);  // [kG8Stages]
  uint64_t* empty = full + kG8Stages;                  // [kG8Stages]
  uint64_t* t_full = empty + kG8Stages;                // [kF8Acc]
  uint64_t* t_empty = t_full + kF8Acc;                 // [kF8Acc]
  uint64_t* f_full = t_empty + kF8Acc;                 // [kF8Ring]
  uint64_t* f_empty = f_full + kF8Ring;                // [kF8Ring]
  unsigned char* stages = smem + 1024;                 // [kG8Stages][weight block 0 | 1 | tokens]
  float* ring = reinterpret_cast<float*>(stages + kG8Stages * static_cast<size_t>(kG8StageBytes));  // [ring][group][tokens]
  float2* ring_w = reinterpret_cast<float2*>(ring + kF8Ring * kF8Group * kG8Tokens);        // [ring][group]
  // GateUp: [tile parity][lane quarter][token] and, per warp, factors; Down: where the tokens' outputs begin
  __shared__ float s_max[MODE == kFp8GateUp ? 2 : 1][4][kG8Tokens];
  __shared__ int64_t s_row[kF8EpiWarps][kG8Tokens / 2];
  __shared__ __align__(16) unsigned char s_out[kF8EpiWarps][2][kG8OutBytes];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  volatile int* abort_flag = &s_abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int kblocks = fp8_blocks(a.k), nblocks = fp8_blocks(a.n);
  if constexpr (MODE == kFp8GateUp) pdl_launch_dependents();  // (a call's last kernel lets nobody ahead)
  if (warp == kF8MmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&s_tmem)),
                 "r"(kF8TmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (tid == 0) {
    for (int i = 0; i < kG8Stages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < kF8Acc; ++i) {
      mbar_init(&t_full[i], 1);
      mbar_init(&t_empty[i], kF8EpiWarps);
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
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  pdl_wait();  // the 8-bit rows, the plan and the scales come from the kernel before
  const int nt = MODE == kFp8GateUp ? nblocks : (nblocks + 1) / 2;  // tiles along the weight rows
  const int mt = MODE == kFp8Linear ? (a.m + a.group - 1) / a.group : __ldcg(a.n_groups);
  const int ntiles = mt * nt;  // (the host refuses more than fit)
  const int step = gridDim.x, step_m = step / nt, step_n = step % nt;
  struct Tile {  // walked without a division per tile: group mi, weight tile ni
    int i, mi, ni;
  };
  auto first_tile = [&]() { return Tile{static_cast<int>(blockIdx.x), static_cast<int>(blockIdx.x) / nt, static_cast<int>(blockIdx.x) % nt}; };
  auto next_tile = [&](Tile t) {
    t.i += step;
    t.mi += step_m;
    t.ni += step_n;
    if (t.ni >= nt) {
      t.ni -= nt;
      ++t.mi;
    }
    return t;
  };
  // A group: expert, first position, tokens. Every role reads its next tile's a tile ahead.
  auto group_of = [&](int mi) {
    if (mi >= mt) return make_int4(0, 0, 0, 0);
    if constexpr (MODE == kFp8Linear) return make_int4(0, mi * a.group, min(a.group, a.m - mi * a.group), 0);
    else return __ldcg(a.groups + mi);
  };
  auto wait = [&](uint64_t* bars, int i, uint32_t parity) {  // a fresh barrier counts as past parity 1
    return f8_wait<false>(smem_addr(bars) + 8 * i, parity, abort_flag, a);
  };
  auto stopped = [&]() { return __any_sync(0xffffffffu, *abort_flag); };

  // Every role is a whole warp that walks the same tiles; one elected lane issues.
  if (warp >= kF8EpiWarps) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kF8RoleRegs));
    Tile next = first_tile();
    int4 ahead = group_of(next.mi);
    if (warp == kF8CopyWarp) {
      // ---- TMA copies --------------------------------------------------------------------------
      int st = 0, past = 1;
      while (next.i < ntiles && !stopped()) {
        const int ni = next.ni;
        const int4 g = ahead;
        next = next_tile(next);
        ahead = group_of(next.mi);
        const int parts = (g.z + kG8Step - 1) / kG8Step;
        const uint32_t bytes = 2 * kF8TileBytes + parts * kG8Step * kFp8Block;
        for (int kb = 0; kb < kblocks; ++kb, (++st == kG8Stages ? (st = 0, past ^= 1) : 0)) {
          if (!wait(empty, st, past)) break;
          if (f8_elect()) {
            unsigned char* sw = stages + static_cast<size_t>(st) * kG8StageBytes;
            const int x = kb * kFp8Block;
            mbar_expect_tx(&full[st], bytes);
            if (MODE == kFp8GateUp) {
              g8_load_weight(sw, &w_map, x, ni * kFp8Block, 0, g.x, &full[st]);
              g8_load_weight(sw + kF8TileBytes, &w_map, x, ni * kFp8Block, 1, g.x, &full[st]);
            } else {
              g8_load_weight(sw, &w_map, x, 2 * ni * kFp8Block, 0, g.x, &full[st]);
              g8_load_weight(sw + kF8TileBytes, &w_map, x, (2 * ni + 1) * kFp8Block, 0, g.x, &full[st]);
            }
            for (int p = 0; p < parts; ++p)
              pt_tma_load_2d(sw + 2 * kF8TileBytes + p * kG8Step * kFp8Block, &x_map, x, g.y + p * kG8Step, &full[st]);
          }
          __syncwarp();
        }
      }
    } else if (warp == kF8MmaWarp) {
      // ---- MMA issuer ----------------------------------------------------------------------------
      int st = 0, ph = 0, buf = 0, past = 1;
      const uint32_t done0 = smem_addr(t_full), freed0 = smem_addr(empty);
      const uint64_t desc0 = pt_desc_sw128(smem_addr(stages));  // + address / 16 within the first 14 bits
      while (next.i < ntiles && !stopped()) {
        const int parts = (ahead.z + kG8Step - 1) / kG8Step;
        next = next_tile(next);
        ahead = group_of(next.mi);
        // fp32 D, e4m3 A and B, K-major, M = 128, N = the tokens in steps of 16
        const uint32_t idesc = (1u << 4) | (static_cast<uint32_t>(parts * kG8Step >> 3) << 17) | (8u << 24);
        for (int kb = 0; kb < kblocks; ++kb) {
          const uint64_t dw = desc0 + static_cast<uint32_t>(st) * (kG8StageBytes >> 4), dx = dw + (2 * kF8TileBytes >> 4);
          const uint32_t d = tmem + 2 * buf * kF8AccCols, done = done0 + 16 * buf;
          if (!wait(full, st, ph) || !wait(t_empty, 2 * buf, past)) break;
          tc_fence_after();
          g8_issue<false>(d, dw, dx, idesc, done, 0);
          if (!wait(t_empty, 2 * buf + 1, past)) break;
          tc_fence_after();
          g8_issue<true>(d + kF8AccCols, dw + (kF8TileBytes >> 4), dx, idesc, done + 8, freed0 + 8 * st);
          if (++st == kG8Stages) {
            st = 0;
            ph ^= 1;
          }
          past ^= buf;
          buf ^= 1;
        }
      }
    } else if (warp == kF8ScaleWarp) {
      // ---- factors: a ring slot's 24 values are loaded together, the next slot's before these are written
      int sl = 0, past = 1;
      while (next.i < ntiles && !stopped()) {
        const int4 g = ahead;
        const int nb0 = MODE == kFp8GateUp ? next.ni : 2 * next.ni;
        const float* sx = a.sx + g.y + lane;
        const float* sw0 = a.ws + (static_cast<int64_t>(g.x) * (MODE == kFp8GateUp ? 2 : 1) * nblocks + nb0) * kblocks;
        // the second block: the up rows' scales, or the next block of columns (none past the last)
        const float* sw1 = MODE == kFp8GateUp ? sw0 + static_cast<int64_t>(nblocks) * kblocks
                                              : (nb0 + 1 < nblocks ? sw0 + kblocks : sw0);
        next = next_tile(next);
        ahead = group_of(next.mi);
        // Where a token's scale goes: the 8 tokens of a unit are four lanes' pairs, a lane's pairs of two
        // units are one 16-byte load, a half of the group begins at 64.
        int at[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int t = lane + 32 * j, c = (g.z + kG8Step - 1) / kG8Step, hf = t >= 8 * c;
          const int u = (t >> 3) - hf * c;  // (past the group: somewhere it never reaches)
          at[j] = t < 2 * 8 * c ? hf * (kG8Tokens / 2) + (u >> 1) * 16 + (t >> 1 & 3) * 4 + (u & 1) * 2 + (t & 1) : -1;
        }
        float s[kF8Group][4];
        float2 w[kF8Group];
        auto load = [&](int kb0) {
#pragma unroll
          for (int i = 0; i < kF8Group; ++i) {
            const bool on = kb0 + i < kblocks;
            const float* p = sx + (kb0 + i) * a.scale_rows;
#pragma unroll
            for (int j = 0; j < 4; ++j) s[i][j] = on && lane + 32 * j < g.z ? __ldcg(p + 32 * j) : 0.f;
            w[i] = on ? make_float2(__ldg(sw0 + kb0 + i), __ldg(sw1 + kb0 + i)) : make_float2(0.f, 0.f);
          }
        };
        load(0);
        for (int kb0 = 0; kb0 < kblocks; kb0 += kF8Group) {
          wait(f_empty, sl, past);
#pragma unroll
          for (int i = 0; i < kF8Group; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (at[j] >= 0) ring[(sl * kF8Group + i) * kG8Tokens + at[j]] = s[i][j];
            if (lane == 0) ring_w[sl * kF8Group + i] = w[i];
          }
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
      int sl = 0, sph = 0, buf = 0, ph = 0;
      uint32_t gone = 0;  // k-blocks of the tiles before this one
      bool given_up = a.wait_ns == 0;
      int kb = 0, b = 0;
      for (int tile = blockIdx.x; tile < ntiles && !given_up; tile += step) {
        for (kb = 0; kb < kblocks; ++kb) {
          if ((kb & (kF8Group - 1)) == 0) {
            wait(f_full, sl, sph);
            if (++sl == kF8Ring) {
              sl = 0;
              sph ^= 1;
            }
          }
#pragma unroll
          for (b = 0; b < 2; ++b) {
            given_up = !wait(t_full, 2 * buf + b, ph);
            if (given_up) break;
#pragma unroll
            for (int p = 0; p < 2; ++p)
              asm volatile("bar.arrive %0, %1;" ::"r"(1 + kF8Acc * p + 2 * buf + b), "n"(32 * 5) : "memory");
          }
          if (given_up) break;
          ph ^= buf;
          buf ^= 1;
        }
        if (!given_up) gone += kblocks;
      }
      if (given_up) {
        const uint32_t first = blockIdx.x, tiles = first < ntiles ? (ntiles - first + step - 1) / step : 0;
        f8_drain<kF8Acc, 32 * 5>(smem_addr(t_empty), a.wait_ns == 0 ? 0 : 2 * (gone + kb) + b, 2 * tiles * kblocks);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kF8EpiRegs));
    // ---- epilogue ------------------------------------------------------------------------------
    const int quarter = warp & 3, hf = warp >> 2;
    const uint32_t lane_base = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    constexpr uint32_t kUpper = 16u << 16;  // the warp's other 16 lanes
    unsigned char(*stage)[kG8OutBytes] = s_out[warp];
    int buf = 0, sl = 0, par = 0;
    // One tile of a group of 16 C tokens, 8 C of them this half's: loads, products and stores of all of
    // them are in flight together (with a bound on every 16 tokens the whole kernel took 1.3 x as long).
    auto tile = [&](auto sixteens, const int4 g, int ni, int2 slots) {
      constexpr int C = decltype(sixteens)::value;
      constexpr bool kAhead = C <= 5;  // an accumulator is loaded while the one before is added (registers)
      constexpr bool kBoth = C <= 6;   // both 16-lane halves are loaded at once
      const int tokens = g.z - hf * 8 * C;  // of this half; may be < 0 or more than 8 C
      uint64_t sum[2][2][C][2];  // [weight block][16-row half][8 tokens][row]: two tokens
#pragma unroll
      for (int i = 0; i < 8 * C; ++i) sum[i / (4 * C)][i / (2 * C) & 1][i / 2 % C][i & 1] = 0;
      float v[2][2][C][4];  // [weight block][half]..
      const uint32_t lane_part = lane_base + hf * 8 * C;
      auto load = [&](auto block, int buf) {
        constexpr int b = decltype(block)::value;
        asm volatile("bar.sync %0, %1;" ::"r"(1 + kF8Acc * hf + 2 * buf + b), "n"(32 * 5) : "memory");
        tc_fence_after();
        const uint32_t d = lane_part + (2 * buf + b) * kF8AccCols;
        g8_ld(d, v[b][0]);
        if (kBoth) g8_ld(d + kUpper, v[b][1]);
      };
      constexpr std::integral_constant<int, 0> b0{};
      constexpr std::integral_constant<int, 1> b1{};
      if (kAhead) load(b0, buf);
      for (int kb = 0; kb < kblocks; ++kb) {
        const int in = kb & (kF8Group - 1);
        if (!kAhead) load(b0, buf);
        const float* f = ring + (sl * kF8Group + in) * kG8Tokens + hf * (kG8Tokens / 2) + 4 * (lane & 3);
        float4 sx[(C + 1) / 2];  // the lane's two tokens of two units of 8
#pragma unroll
        for (int c = 0; c < (C + 1) / 2; ++c) sx[c] = *reinterpret_cast<const float4*>(f + 16 * c);
        const float2 sw = ring_w[sl * kF8Group + in];
        auto add = [&](auto block, int h) {
          constexpr int b = decltype(block)::value;
          const float w = b ? sw.y : sw.x;
#pragma unroll
          for (int c = 0; c < C; ++c) {
            const float4 s = sx[c >> 1];
            const uint64_t f = g8_mul(c & 1 ? g8_pair(s.z, s.w) : g8_pair(s.x, s.y), g8_pair(w, w));
            const float(&u)[4] = v[b][h][c];
            uint64_t(&o)[2] = sum[b][h][c];
            o[0] = g8_fma(g8_pair(u[0], u[1]), f, o[0]);
            o[1] = g8_fma(g8_pair(u[2], u[3]), f, o[1]);
          }
        };
        auto loaded = [&](auto block) {  // the accumulator is in registers: it may be written again
          constexpr int b = decltype(block)::value;
          g8_ld_wait(v[b][0]);
          if (kBoth) {
            g8_ld_wait(v[b][1]);
          } else {
            add(block, 0);
            g8_ld(lane_part + (2 * buf + b) * kF8AccCols + kUpper, v[b][1]);
            g8_ld_wait(v[b][1]);
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&t_empty[2 * buf + b]);
        };
        loaded(b0);
        if (kAhead) load(b1, buf);
        if (kBoth) add(b0, 0);
        add(b0, 1);
        if (!kAhead) load(b1, buf);
        loaded(b1);
        buf ^= 1;
        if (in == kF8Group - 1 || kb == kblocks - 1) {  // the group's factors are read
          if (lane == 0) mbar_arrive(&f_empty[sl]);
          if (++sl == kF8Ring) sl = 0;
        }
        if (kAhead && kb + 1 < kblocks) load(b0, buf);
        if (kBoth) add(b1, 0);
        add(b1, 1);
      }
      if constexpr (MODE == kFp8GateUp) {
        // h, and its maximum per token: over this lane's 4 rows, then over the 8 lanes of the same
        // tokens; in the first step a lane hands over the half that it does not keep.
        float biggest[2 * C];  // [8 tokens][token]
#pragma unroll
        for (int i = 0; i < 4 * C; ++i) {  // rows past I have zero weights: h = 0
          const int h = i / (2 * C), c = i / 2 % C;
          uint64_t& v = sum[0][h][c][i & 1];
          v = g8_silu_mul(v, sum[1][h][c][i & 1]);
          const float2 t = g8_unpair(v);
          float* m = &biggest[2 * c];
          m[0] = g8_max_abs(h || (i & 1) ? m[0] : 0.f, t.x);
          m[1] = g8_max_abs(h || (i & 1) ? m[1] : 0.f, t.y);
        }
        uint32_t most[2 * C];
#pragma unroll
        for (int i = 0; i < 2 * C; ++i) most[i] = __float_as_uint(biggest[i]);
        // each lane of a pair hands over the half that it does not keep
        constexpr int kHalf = C % 2 == 0 ? C / 2 : C;  // kept after the second step (an odd C: everything)
        const bool up = lane & 16, up2 = C % 2 == 0 && (lane & 8);
#pragma unroll
        for (int i = 0; i < C; ++i)
          most[i] = max(up ? most[i + C] : most[i], __shfl_xor_sync(0xffffffffu, up ? most[i] : most[i + C], 16));
#pragma unroll
        for (int i = 0; i < kHalf; ++i) {
          constexpr int kOther = C % 2 == 0 ? C / 2 : 0;
          uint32_t m = max(up2 ? most[i + kOther] : most[i], __shfl_xor_sync(0xffffffffu, up2 ? most[i] : most[i + kOther], 8));
          m = max(m, __shfl_xor_sync(0xffffffffu, m, 4));
          const int k = (up ? C : 0) + (up2 ? kHalf : 0) + i;  // of 2 C
          if ((lane & 4) == 0 && (C % 2 == 0 || (lane & 8) == 0))
            s_max[par][quarter][hf * 64 + (k >> 1) * 8 + 2 * (lane & 3) + (k & 1)] = __uint_as_float(m);
        }
        asm volatile("bar.sync %0, 128;" ::"r"(1 + 2 * kF8Acc + hf) : "memory");  // the four quarters of this half
        float* fac = reinterpret_cast<float*>(s_row[warp]);
#pragma unroll
        for (int t = lane; t < 8 * C; t += 32) {
          uint32_t m = 0;
#pragma unroll
          for (int q = 0; q < 4; ++q) m = max(m, __float_as_uint(s_max[par][q][hf * 64 + t]));
          const float am = fp8_amax(m);
          fac[t] = kE4m3Max / am;
          if (quarter == 0 && t < tokens) a.hs[ni * a.scale_rows + g.y + hf * 8 * C + t] = am / kE4m3Max;
        }
        __syncwarp();
        // 16-bit elements (row, row + 8), transposed through shared memory: 32 bytes a token (and 16
        // against bank conflicts), of which a lane takes 16 and puts its 16 rows in order.
        const int64_t pitch = f8_row_pitch(a.n);
        uint8_t* dst = a.hq + static_cast<int64_t>(g.y + hf * 8 * C + lane / 2) * pitch + ni * kFp8Block + quarter * 32 +
                       (lane & 1) * 16;
        const int to = ((lane >> 4) * 8 + (lane & 7)) * 48 + (lane >> 3 & 1) * 16;
#pragma unroll
        for (int c = 0; c < C; c += 2) {
          uint32_t q[4];  // [8 tokens][16-row half]
#pragma unroll
          for (int i = 0; i < (c + 1 < C ? 4 : 2); ++i) {
            const float2 f = *reinterpret_cast<const float2*>(fac + (c + (i >> 1)) * 8 + 2 * (lane & 3));
            const uint64_t(&u)[2] = sum[0][i & 1][c + (i >> 1)];
            const float2 lo = g8_unpair(g8_mul(u[0], g8_pair(f.x, f.y))), hi = g8_unpair(g8_mul(u[1], g8_pair(f.x, f.y)));
            q[i] = e4m3x4(lo.x, hi.x, lo.y, hi.y);
          }
          unsigned char* out = stage[c >> 1 & 1];
          if (c + 1 < C) g8_store_matrices(out + to, q[0], q[1], q[2], q[3]);
          else g8_store_matrices(out + to, q[0], q[1]);
          __syncwarp();
          const uint4 u = *reinterpret_cast<const uint4*>(out + (lane / 2) * 48 + (lane & 1) * 16);
          if (8 * c + lane / 2 < tokens && (c + 1 < C || lane < 16))
            *reinterpret_cast<uint4*>(dst + 8 * c * pitch) =
                make_uint4(__byte_perm(u.x, u.y, 0x6420), __byte_perm(u.z, u.w, 0x6420), __byte_perm(u.x, u.y, 0x7531),
                           __byte_perm(u.z, u.w, 0x7531));
        }
        par ^= 1;
      } else {
        float acc[2][2][C][4];  // [weight block][16-row half][8 tokens][2 row + token]
  #pragma unroll
        for (int i = 0; i < 8 * C; ++i) {
          const float2 t = g8_unpair(sum[i / (4 * C)][i / (2 * C) & 1][i / 2 % C][i & 1]);
          float* p = &acc[i / (4 * C)][i / (2 * C) & 1][i / 2 % C][2 * (i & 1)];
          p[0] = t.x;
          p[1] = t.y;
        }
        int64_t* off = s_row[warp];
        __syncwarp();
#pragma unroll
        for (int t = 0; t < (C > 4 ? 2 : 1); ++t) {
          if constexpr (MODE == kFp8Linear) {
            off[lane + 32 * t] = static_cast<int64_t>(g.y + hf * 8 * C + lane + 32 * t) * a.out_stride;
          } else {
            const int slot = t ? slots.y : slots.x, q = slot / a.s;
            off[lane + 32 * t] = q * a.out_stride + (slot - q * a.s) * a.out_stride_s;
          }
        }
        __syncwarp();
        const int have = min(tokens, 8 * C);
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const int col = (2 * ni + b) * kFp8Block + quarter * 32, n = a.n - col;
          if (n <= 0) continue;
          const bool vec = a.out_vec && n >= 32;
          auto store = [&](auto* out) {
            using TO = std::remove_pointer_t<decltype(out)>;
            if (vec) g8_store<TO, true>(out + col, n, acc[b], off, stage, have, lane);
            else g8_store<TO, false>(out + col, n, acc[b], off, stage, have, lane);
          };
          if (a.out_dtype == ALUT_BF16) store(static_cast<__nv_bfloat16*>(a.out));
          else if (a.out_dtype == ALUT_F16) store(static_cast<__half*>(a.out));
          else g8_store<float, false>(static_cast<float*>(a.out) + col, n, acc[b], off, stage, have, lane);
        }
      }
    };
    Tile next = first_tile();
    int4 ahead = group_of(next.mi);
    while (next.i < ntiles) {
      const int ni = next.ni;
      const int4 g = ahead;
      next = next_tile(next);
      ahead = group_of(next.mi);
      int2 slots = make_int2(0, 0);  // Down: those of this lane's tokens (past the group: any)
      if (MODE == kFp8Down) {
        const int at = hf * 8 * ((g.z + kG8Step - 1) / kG8Step) + lane;
        if (at < g.z) slots.x = __ldcg(a.sorted + g.y + at);
        if (at + 32 < g.z) slots.y = __ldcg(a.sorted + g.y + at + 32);
      }
      switch ((g.z + kG8Step - 1) / kG8Step) {
        case 1: tile(std::integral_constant<int, 1>{}, g, ni, slots); break;
        case 2: tile(std::integral_constant<int, 2>{}, g, ni, slots); break;
        case 3: tile(std::integral_constant<int, 3>{}, g, ni, slots); break;
        case 4: tile(std::integral_constant<int, 4>{}, g, ni, slots); break;
        case 5: tile(std::integral_constant<int, 5>{}, g, ni, slots); break;
        case 6: tile(std::integral_constant<int, 6>{}, g, ni, slots); break;
        case 7: tile(std::integral_constant<int, 7>{}, g, ni, slots); break;
        default: tile(std::integral_constant<int, 8>{}, g, ni, slots); break;
      }
    }
  }

  __syncthreads();
  if (*abort_flag && tid == 0) {  // what is in flight gets 10 ms to end before the memory goes
    const uint64_t t0 = global_ns();
    while (global_ns() - t0 < 10000000ull) __nanosleep(1000);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kF8MmaWarp)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kF8TmemCols) : "memory");
}

}  // namespace alut
