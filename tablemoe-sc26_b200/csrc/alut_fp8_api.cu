// C ABI of the 8-bit products (alut_quantize_fp8, alut_linear_fp8, alut_experts_fp8 of
// include/alut.h): argument checks on the host, workspace layout, kernel choice, launches.
#include <algorithm>

#include "alut_fp8.cuh"
#include "alut_fp8_grouped.cuh"
#include "alut_fp8_tc.cuh"
#include "alut_host.cuh"

namespace alut {

static thread_local uint64_t g_wait_ns = kWaitNs;  // alut_set_wait_limit

static int64_t round_up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

// Checks shared by every e4m3 weight.
static int check_weight(const char* what, const void* w, const float* scale, int64_t row_stride, int k) {
  if (!w || !scale) return fail(ALUT_EINVAL, "%s: NULL weight or scale", what);
  if (!aligned16(w) || row_stride % 16 != 0)
    return fail(ALUT_ESHAPE, "%s: weight rows must be 16-byte aligned (row stride %lld)", what,
                static_cast<long long>(row_stride));
  if (row_stride < round_up(k, 16))
    return fail(ALUT_ESHAPE, "%s: weight row stride %lld < %lld", what, static_cast<long long>(row_stride),
                static_cast<long long>(round_up(k, 16)));
  return ALUT_OK;
}

static bool rows_vec(const void* x, int64_t stride, int dtype) {
  return aligned16(x) && (stride * dtype_size(dtype)) % 16 == 0;
}

template <int MODE>
static int launch_stream(StreamArgs a, int x_dtype, unsigned groups, bool pdl, cudaStream_t st) {
  const int rows = MODE == kFp8GateUp ? kStreamWRows : 2 * kStreamWRows;  // of a row group
  const int kblocks = fp8_blocks(a.k);
  auto slices = [&](int ks, int steps) {
    return static_cast<int64_t>(ceil_div(a.n, static_cast<int64_t>(steps) * (kStreamWarps / ks) * rows));
  };
  // Few CTAs: every warp a share of K, the shortest way through. Two for each SM (whether or not two
  // fit, above K = 3840 one does): at least 3
  // k-blocks a warp and up to kStreamMaxSteps steps per CTA, over which the search for the group and
  // x's form are paid once. Measured, 8 rows: 32000 x 2048 19.2 us with this and 25.3 with all warps
  // across K, 150000 x 2048 59 and 96 (71 with one step per CTA); up to 12288 x 2048 there is no difference.
  a.steps = 1;
  int ks = kStreamWarps;
  while (ks > kblocks) ks /= 2;
  int wide = ks;
  while (wide > 1 && kblocks < 3 * wide) wide /= 2;
  if (groups * slices(wide, 1) >= 2 * num_sms()) {
    ks = wide;
    while (a.steps < kStreamMaxSteps && groups * slices(wide, a.steps + 1) >= 4 * num_sms()) ++a.steps;
  }
  for (a.lks = 0; (1 << a.lks) < ks;) ++a.lks;
  const dim3 grid(groups, static_cast<unsigned>(slices(ks, a.steps)));
  if (grid.y > 65535u) return fail(ALUT_ERANGE, "fp8: %d weight rows", a.n);
  const dim3 block(32 * kStreamWarps);
  void (*kern)(StreamArgs) = nullptr;
  if (MODE == kFp8Down || x_dtype == ALUT_F32) kern = k_fp8_stream<float, MODE>;
  if constexpr (MODE != kFp8Down) {
    if (x_dtype == ALUT_BF16) kern = k_fp8_stream<__nv_bfloat16, MODE>;
    if (x_dtype == ALUT_F16) kern = k_fp8_stream<__half, MODE>;
  }
  const size_t smem = stream_smem_bytes(a.k, a.steps, ks);
  // (with the kernel's static shared memory the default limit is reached below 48 KB)
  const int rc = allow_smem(reinterpret_cast<const void*>(kern), std::max<size_t>(smem, 64 * 1024));
  if (rc) return rc;
  if (!pdl) {
    kern<<<grid, block, smem, st>>>(a);
    return check_launch("k_fp8_stream");
  }
  const cudaError_t e = launch_pdl(kern, grid, block, smem, st, a);
  if (e != cudaSuccess) return fail(ALUT_ECUDA, "k_fp8_stream: %s", cudaGetErrorString(e));
  return ALUT_OK;
}

// TMA map of a byte tensor of up to 4 dimensions (strides in bytes of dimensions 1..): boxes of
// 128 bytes x box_rows rows with the 128-byte swizzle, out-of-range parts read as zeros.
static int encode_map(CUtensorMap* map, const void* p, int nd, const uint64_t* dims, const uint64_t* strides,
                      uint32_t box_rows) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static Encode encode = nullptr;
  if (!encode) {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult qr{};
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &qr) != cudaSuccess ||
        qr != cudaDriverEntryPointSuccess || !fn)
      return fail(ALUT_ECUDA, "cuTensorMapEncodeTiled is not available");
    encode = reinterpret_cast<Encode>(fn);
  }
  cuuint64_t d[4], st[3];
  const cuuint32_t box[4] = {kFp8Block, box_rows, 1, 1}, estr[4] = {1, 1, 1, 1};
  for (int i = 0; i < nd; ++i) d[i] = dims[i];
  for (int i = 0; i + 1 < nd; ++i) st[i] = strides[i];
  const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, nd, const_cast<void*>(p), d, st, box, estr,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(ALUT_ECUDA, "cuTensorMapEncodeTiled: error %d", static_cast<int>(r));
  return ALUT_OK;
}

// 8-bit rows [rows][f8_row_pitch(k)].
static int encode_rows(CUtensorMap* map, const void* p, int64_t rows, int k, uint32_t box_rows) {
  const uint64_t dims[2] = {static_cast<uint64_t>(f8_row_pitch(k)), static_cast<uint64_t>(rows)};
  const uint64_t strides[1] = {static_cast<uint64_t>(f8_row_pitch(k))};
  return encode_map(map, p, 2, dims, strides, box_rows);
}

// A weight [experts][halves][rows][k]; a dimension of extent 1 takes any stride.
static int encode_weight(CUtensorMap* map, const void* p, int k, int rows, int halves, int experts, int64_t row_stride,
                         int64_t half_stride, int64_t expert_stride) {
  const uint64_t any = static_cast<uint64_t>(row_stride);
  const uint64_t dims[4] = {static_cast<uint64_t>(k), static_cast<uint64_t>(rows), static_cast<uint64_t>(halves),
                            static_cast<uint64_t>(experts)};
  const uint64_t strides[3] = {static_cast<uint64_t>(row_stride), halves > 1 ? static_cast<uint64_t>(half_stride) : any,
                               experts > 1 ? static_cast<uint64_t>(expert_stride) : any};
  return encode_map(map, p, 4, dims, strides, kF8Rows);
}

static int launch_tc(const CUtensorMap& xm, const CUtensorMap& wm, const F8Args& a, int64_t max_tiles, cudaStream_t st) {
  const int rc = allow_smem(reinterpret_cast<const void*>(k_fp8_tc), kF8SmemBytes);
  if (rc) return rc;
  if (max_tiles + num_sms() > 0x7fffffffll) return fail(ALUT_ERANGE, "fp8: %lld tiles", static_cast<long long>(max_tiles));
  const unsigned grid = 2 * static_cast<unsigned>(std::min<int64_t>(max_tiles, num_sms() / 2));  // pairs of CTAs
  const cudaError_t e = launch_pdl(k_fp8_tc, dim3(grid), dim3(kF8Threads), kF8SmemBytes, st, xm, wm, a);
  if (e != cudaSuccess) return fail(ALUT_ECUDA, "k_fp8_tc: %s", cudaGetErrorString(e));
  return ALUT_OK;
}

template <int MODE>
static int launch_grouped(const CUtensorMap& xm, const CUtensorMap& wm, const F8Args& a, int64_t max_tiles, cudaStream_t st) {
  auto kern = k_fp8_grouped<MODE>;
  const int rc = allow_smem(reinterpret_cast<const void*>(kern), kG8SmemBytes);
  if (rc) return rc;
  if (max_tiles + num_sms() > 0x7fffffffll) return fail(ALUT_ERANGE, "fp8: %lld tiles", static_cast<long long>(max_tiles));
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(max_tiles, num_sms()));
  const cudaError_t e = launch_pdl(kern, dim3(grid), dim3(kF8Threads), kG8SmemBytes, st, xm, wm, a);
  if (e != cudaSuccess) return fail(ALUT_ECUDA, "k_fp8_grouped: %s", cudaGetErrorString(e));
  return ALUT_OK;
}

static int launch_rows(const F8PrepArgs& a, int x_dtype, cudaStream_t st) {
  const int64_t units = static_cast<int64_t>(a.rows) * ceil_div(fp8_blocks(a.k), kF8RowBlocks);
  if (units + 8 > 0x7fffffffll) return fail(ALUT_ERANGE, "fp8: %d rows of %d columns", a.rows, a.k);
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>((units + 7) / 8, kF8RowCtas * num_sms()));
  auto kern = x_dtype == ALUT_BF16 ? k_fp8_rows<__nv_bfloat16> : x_dtype == ALUT_F16 ? k_fp8_rows<__half> : k_fp8_rows<float>;
  if (!a.place) {
    kern<<<grid, 256, 0, st>>>(a);
    return check_launch("k_fp8_rows");
  }
  const cudaError_t e = launch_pdl(kern, dim3(grid), dim3(256), 0, st, a);
  if (e != cudaSuccess) return fail(ALUT_ECUDA, "k_fp8_rows: %s", cudaGetErrorString(e));
  return ALUT_OK;
}

// Which product a call takes. The streaming one reads the weights once per 8 rows, the tensor-core ones
// from L2 once per group, after a launch that writes x's 8-bit form. Measured (us, streaming / tensor cores,
// weights from HBM): 2048 x 2048 5.6 / 12.7 for 1 row, 6.8 / 12.9 for 32, 12.0 / 14.7 for 64; 4096 x 4096
// 10.2 / 18.7 for 1, 15.3 / 18.7 for 16, 21.7 / 18.8 for 24; 2560 x 2560 12.4 / 14.3 for 32, 15.3 / 16.7 for
// 64; 12288 x 2048 12.2 / 13.9 for 8, 16.4 / 14.0 for 24; 150000 x 2048 61 / 83 for 8, 88 / 80 for 16: what is
// read in all decides, and one pass is always streamed. Where that is little, the passes over x's form
// do: 1024 x 1024 7.4 / 10.7 for 128, 10.4 / 10.7 for 192, 13.1 / 10.6 for 256; 2048 x 768 9.4 / 9.7 for 128,
// 11.0 / 9.8 for 192. Past kStreamMaxBlocks x's words do not fit beside the ring, and few rows are left with
// one group's ceil(n / 256) CTAs: 4096 x 8192 18.1 us for 1 row, x 8320 29.1, x 12288 40.4.
static bool linear_streams(int m, int n, int k) {
  const int64_t passes = ceil_div(m, kStreamRows);
  return (passes == 1 || (passes <= 16 && passes * n * k <= (40ll << 20))) && fp8_blocks(k) <= kStreamMaxBlocks;
}
// Tokens to a group of the grouped kernel, as few as still make one tile per SM; 0: pairs of CTAs, once
// their tiles of 256 x 256 occupy about half the GPU. Measured (us, grouped / pairs): 2560 x 2560 14.2 /
// 18.0 for 512 rows, 16.9 / 18.6 for 1024, 40.9 / 32.1 for 2048; 4096 x 4096 17.3 / 23.3 for 136, 20.5 / 24.2 for
// 512, 26.2 / 24.8 for 768, 219 / 171 for 8192; 12288 x 2048 12.4 / 15.8 for 64, 17.1 / 16.7 for 256; 768 x
// 2048 14.0 / 16.6 for 2048, 40.9 / 33.6 for 8192.
static int linear_group(int m, int n) {
  const int tiles = (fp8_blocks(n) + 1) / 2;
  if (static_cast<int64_t>(ceil_div(m, kG8Tokens)) * tiles > 64) return 0;
  const int groups = std::max(1, num_sms() / tiles);
  return std::min<int>(kG8Tokens, static_cast<int>(round_up(ceil_div(m, groups), kG8Step)));
}
// The same for routed slots, where the streaming kernels save the plan and the pass over x: 8 slots of
// 128 experts of 2048 x 768 24.6 / 25.9 us, of 24 of 1000 x 600 17.2 / 20.0, of 8 of 2048 x 2816 34.0 / 31.8;
// but 32 slots 51.9 / 47.3, 23.9 / 22.1, 50.5 / 45.1 and 128 slots 98 / 83, 35.5 / 25.8, 120 / 48.
static bool experts_stream(const alut_fp8_experts_t* ex, int64_t slots) {
  return slots <= kStreamMaxSlots && fp8_blocks(std::max(ex->h, ex->i)) <= kStreamMaxBlocks;
}

// Tokens to a group at most, by the mean of the experts' slots: groups of one size fill the SMs evenly where a
// few experts have most of the slots, but each reads its expert's weights again. Measured (us, groups of up
// to 48 / 64 / 96 / 128, experts drawn unevenly), 128 experts of 2048 x 768: 32 slots each 131 / 135 / 142 / 144,
// 64 154 / 147 / 156 / 166, 96 203 / 190 / 183 / 194, 192 342 / 312 / 294 / 286; 72 of 2560 x 1280: 32 139 / 138 /
// 142 / 146, 128 246 / 245 / 216 / 235, 192 386 / 340 / 310 / 305; 24 of 1000 x 600: 32 25.9 / 26.8 / 27.9 / 32.5.
static int experts_group(const alut_fp8_experts_t* ex, int64_t slots) {
  const int64_t mean = slots / ex->num_experts;
  return mean > 160 ? kG8Tokens : static_cast<int>(round_up(std::min<int64_t>(std::max<int64_t>(mean, 48), 96), kG8Step));
}

struct LinearWorkspace {
  size_t xq, sx, total;
};
static LinearWorkspace linear_layout(int m, int n, int k) {
  LinearWorkspace w{};
  size_t off = 0;
  if (!linear_streams(m, n, k)) {
    w.xq = off; off = align256(off + static_cast<size_t>(m) * f8_row_pitch(k));
    w.sx = off; off = align256(off + sizeof(float) * m * fp8_blocks(k));
  }
  w.total = off;
  return w;
}

// Workspace of alut_experts_fp8, in order; every part starts on 256 bytes.
struct ExpertsWorkspace {
  size_t n_groups, groups, sorted, place, xq, sx, hidden, hs, total;
  int64_t max_groups;
};
static ExpertsWorkspace experts_layout(const alut_fp8_experts_t* ex, int q, int s) {
  ExpertsWorkspace w{};
  const int64_t n = static_cast<int64_t>(q) * s;
  size_t off = 0;
  if (experts_stream(ex, n)) {
    w.hidden = off; off = align256(off + sizeof(float) * n * round_up(ex->i, 4));
  } else {
    w.max_groups = ceil_div(n, experts_group(ex, n)) + std::min<int64_t>(n, ex->num_experts);
    w.n_groups = off; off = align256(off + sizeof(int));
    w.groups = off;   off = align256(off + sizeof(int4) * w.max_groups);
    w.sorted = off;   off = align256(off + sizeof(int) * n);
    w.place = off;    off = align256(off + sizeof(int) * n);
    w.xq = off;       off = align256(off + static_cast<size_t>(n) * f8_row_pitch(ex->h));
    w.sx = off;       off = align256(off + sizeof(float) * n * fp8_blocks(ex->h));
    w.hidden = off;   off = align256(off + static_cast<size_t>(n) * f8_row_pitch(ex->i));
    w.hs = off;       off = align256(off + sizeof(float) * n * fp8_blocks(ex->i));
  }
  w.total = off;
  return w;
}

static int check_experts(const alut_fp8_experts_t* ex) {
  if (!ex) return fail(ALUT_EINVAL, "experts is NULL");
  if (ex->num_experts <= 0 || ex->h <= 0 || ex->i <= 0)
    return fail(ALUT_EINVAL, "experts: num_experts=%d h=%d i=%d must be positive", ex->num_experts, ex->h, ex->i);
  if (ex->num_experts > kFp8MaxExperts)
    return fail(ALUT_ERANGE, "experts: num_experts=%d exceeds %d", ex->num_experts, kFp8MaxExperts);
  int rc = check_weight("experts gate_up", ex->gate_up, ex->gate_up_scale, ex->gate_up_stride[2], ex->h);
  if (rc) return rc;
  rc = check_weight("experts down", ex->down, ex->down_scale, ex->down_stride[1], ex->i);
  if (rc) return rc;
  if (ex->gate_up_stride[0] % 16 != 0 || ex->gate_up_stride[1] % 16 != 0 || ex->down_stride[0] % 16 != 0 ||
      ex->gate_up_stride[0] < 0 || ex->gate_up_stride[1] < 0 || ex->down_stride[0] < 0)
    return fail(ALUT_ESHAPE, "experts: strides must be multiples of 16 bytes");
  return ALUT_OK;
}

}  // namespace alut

using namespace alut;

extern "C" {

int alut_quantize_fp8(int64_t batch, int64_t rows, int32_t cols, int32_t block_rows, const void* src, int32_t dtype,
                      int64_t src_stride_b, int64_t src_stride, void* out, int64_t out_stride_b, int64_t out_stride,
                      float* scale, alut_stream_t stream) {
  if (batch < 0 || rows < 0 || cols < 0) return fail(ALUT_EINVAL, "quantize_fp8: negative size");
  if (block_rows != 1 && block_rows != kFp8Block)
    return fail(ALUT_EINVAL, "quantize_fp8: block_rows=%d must be 1 or %d", block_rows, kFp8Block);
  if (!dtype_ok(dtype)) return fail(ALUT_EDTYPE, "quantize_fp8: dtype");
  if (batch == 0 || rows == 0 || cols == 0) return ALUT_OK;
  if (!src || !out || !scale) return fail(ALUT_EINVAL, "quantize_fp8: NULL argument");
  if (src_stride < cols || out_stride < cols) return fail(ALUT_ESHAPE, "quantize_fp8: row strides");
  QuantArgs a{batch, rows, cols, src, src_stride_b, src_stride, static_cast<uint8_t*>(out), out_stride_b,
              out_stride, scale};
  a.src_vec = rows_vec(src, src_stride, dtype) && rows_vec(src, src_stride_b, dtype);
  a.out_vec = (reinterpret_cast<uintptr_t>(out) | out_stride | out_stride_b) % 8 == 0;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int64_t kb = fp8_blocks(cols);
  if (block_rows == 1) {
    const int64_t n = batch * rows * ((kb + kQuantBlocks - 1) / kQuantBlocks);
    auto kern = dtype == ALUT_BF16 ? k_fp8_quantize_rows<__nv_bfloat16>
                                   : dtype == ALUT_F16 ? k_fp8_quantize_rows<__half> : k_fp8_quantize_rows<float>;
    kern<<<static_cast<unsigned>(std::min<int64_t>((n + 7) / 8, 16 * num_sms())), 256, 0, st>>>(a);
    return check_launch("k_fp8_quantize_rows");
  }
  const int64_t n = batch * ((rows + kFp8Block - 1) / kFp8Block) * kb;
  auto kern = dtype == ALUT_BF16 ? k_fp8_quantize_blocks<__nv_bfloat16>
                                 : dtype == ALUT_F16 ? k_fp8_quantize_blocks<__half> : k_fp8_quantize_blocks<float>;
  kern<<<static_cast<unsigned>(std::min<int64_t>(n, 1 << 20)), 256, 0, st>>>(a);
  return check_launch("k_fp8_quantize_blocks");
}

int alut_set_wait_limit(uint64_t ns) {
  g_wait_ns = ns;
  return ALUT_OK;
}

size_t alut_linear_fp8_workspace_size(int32_t m, int32_t n, int32_t k) {
  if (m < 0 || n <= 0 || k <= 0) return 0;
  return linear_layout(m, n, k).total;
}

int alut_linear_fp8(int32_t m, int32_t n, int32_t k, const void* x, int32_t x_dtype, int64_t x_stride, const void* w,
                    int64_t w_stride, const float* w_scale, void* out, int32_t out_dtype, int64_t out_stride,
                    uint32_t* error_bits, void* workspace, size_t workspace_bytes, alut_stream_t stream) {
  if (m < 0 || n <= 0 || k <= 0) return fail(ALUT_EINVAL, "linear_fp8: m=%d n=%d k=%d", m, n, k);
  if (!dtype_ok(x_dtype) || !dtype_ok(out_dtype)) return fail(ALUT_EDTYPE, "linear_fp8: dtype");
  if (m == 0) return ALUT_OK;
  if (!x || !out) return fail(ALUT_EINVAL, "linear_fp8: NULL argument");
  if (x_stride < k || out_stride < n) return fail(ALUT_ESHAPE, "linear_fp8: strides");
  int rc = check_weight("linear_fp8", w, w_scale, w_stride, k);
  if (rc) return rc;
  const size_t need = alut_linear_fp8_workspace_size(m, n, k);
  if ((need && !workspace) || workspace_bytes < need)
    return fail(ALUT_EWORKSPACE, "linear_fp8: workspace has %zu bytes, needs %zu", workspace_bytes, need);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (!linear_streams(m, n, k)) {
    if (!aligned16(workspace)) return fail(ALUT_EWORKSPACE, "linear_fp8: workspace must be 16-byte aligned");
    const LinearWorkspace ws = linear_layout(m, n, k);
    char* base = static_cast<char*>(workspace);
    F8PrepArgs p{};
    p.x = x;
    p.x_stride = x_stride;
    p.rows = m;
    p.k = k;
    p.x_vec = rows_vec(x, x_stride, x_dtype);
    p.xq = reinterpret_cast<uint8_t*>(base + ws.xq);
    p.sx = reinterpret_cast<float*>(base + ws.sx);
    p.scale_rows = m;
    CUtensorMap xm, wm;
    const int group = linear_group(m, n);
    rc = encode_rows(&xm, p.xq, m, k, group ? kG8Step : kF8Rows);
    if (!rc && group) {
      rc = encode_weight(&wm, w, k, n, 1, 1, w_stride, 0, 0);
    } else if (!rc) {
      const uint64_t dims[2] = {static_cast<uint64_t>(k), static_cast<uint64_t>(n)}, strides[1] = {static_cast<uint64_t>(w_stride)};
      rc = encode_map(&wm, w, 2, dims, strides, kF8Rows);
    }
    if (!rc) rc = launch_rows(p, x_dtype, st);
    if (rc) return rc;
    F8Args a{};
    a.m = m;
    a.n = n;
    a.k = k;
    a.sx = p.sx;
    a.scale_rows = m;
    a.ws = w_scale;
    a.out = out;
    a.out_dtype = out_dtype;
    a.out_stride = out_stride;
    a.out_vec = rows_vec(out, out_stride, out_dtype);
    a.err = error_bits;
    a.wait_ns = g_wait_ns;
    a.group = group;
    if (group) return launch_grouped<kFp8Linear>(xm, wm, a, static_cast<int64_t>(ceil_div(m, group)) * ((fp8_blocks(n) + 1) / 2), st);
    return launch_tc(xm, wm, a, static_cast<int64_t>(ceil_div(m, kF8PairRows)) * ((fp8_blocks(n) + 1) / 2), st);
  }
  StreamArgs a{};
  a.x = x;
  a.x_stride = x_stride;
  a.x_vec = rows_vec(x, x_stride, x_dtype);
  a.m = m;
  a.n = n;
  a.k = k;
  a.w = static_cast<const uint8_t*>(w);
  a.w_stride = w_stride;
  a.ws = w_scale;
  a.out = out;
  a.out_dtype = out_dtype;
  a.out_stride = out_stride;
  return launch_stream<kFp8Linear>(a, x_dtype, static_cast<unsigned>(ceil_div(m, kStreamRows)), false, st);
}

size_t alut_experts_fp8_workspace_size(const alut_fp8_experts_t* ex, int32_t q, int32_t s) {
  if (!ex || ex->num_experts <= 0 || ex->i <= 0 || ex->h <= 0 || q < 0 || s < 0 || s > kMaxSlots) return 0;
  if (static_cast<int64_t>(q) * s >= (1ll << 31)) return 0;
  return experts_layout(ex, q, s).total;
}

int alut_experts_fp8(const alut_fp8_experts_t* ex, int32_t q, int32_t s, const void* x, int32_t x_dtype,
                     int64_t x_stride, const int64_t* sel, int64_t sel_stride, const uint8_t* compute,
                     int64_t compute_stride, int32_t zero_skipped, void* out, int32_t out_dtype, int64_t out_stride_t,
                     int64_t out_stride_s, uint32_t* error_bits, void* workspace, size_t workspace_bytes,
                     alut_stream_t stream) {
  int rc = check_experts(ex);
  if (rc) return rc;
  if (q < 0 || s < 0) return fail(ALUT_EINVAL, "experts_fp8: q=%d s=%d", q, s);
  if (s > kMaxSlots) return fail(ALUT_ERANGE, "experts_fp8: s=%d exceeds %d", s, kMaxSlots);
  if (static_cast<int64_t>(q) * s >= (1ll << 31)) return fail(ALUT_ERANGE, "experts_fp8: q*s too large");
  if (!dtype_ok(x_dtype) || !dtype_ok(out_dtype)) return fail(ALUT_EDTYPE, "experts_fp8: dtype");
  if (q == 0 || s == 0) return ALUT_OK;
  if (!x || !sel || !out) return fail(ALUT_EINVAL, "experts_fp8: NULL argument");
  if (x_stride < ex->h || sel_stride < s || (compute && compute_stride < s) || out_stride_s < ex->h ||
      out_stride_t < ex->h)
    return fail(ALUT_ESHAPE, "experts_fp8: strides");
  const ExpertsWorkspace ws = experts_layout(ex, q, s);
  if (!workspace || workspace_bytes < ws.total)
    return fail(ALUT_EWORKSPACE, "experts_fp8: workspace has %zu bytes, needs %zu", workspace_bytes, ws.total);
  if (!aligned16(workspace)) return fail(ALUT_EWORKSPACE, "experts_fp8: workspace must be 16-byte aligned");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  char* base = static_cast<char*>(workspace);
  const int n = q * s;
  Fp8Route r{q, s, ex->num_experts, sel, sel_stride, compute, compute_stride,
             sel_stride == s && (!compute || compute_stride == s), error_bits};
  if (!experts_stream(ex, n)) {
    F8PrepArgs p{};
    p.x = x;
    p.x_stride = x_stride;
    p.rows = q;
    p.k = ex->h;
    p.x_vec = rows_vec(x, x_stride, x_dtype);
    p.xq = reinterpret_cast<uint8_t*>(base + ws.xq);
    p.sx = reinterpret_cast<float*>(base + ws.sx);
    p.scale_rows = n;
    p.place = reinterpret_cast<int*>(base + ws.place);
    p.s = s;
    p.out = zero_skipped ? out : nullptr;
    p.out_dtype = out_dtype;
    p.out_vec = rows_vec(out, out_stride_t, out_dtype) && rows_vec(out, out_stride_s, out_dtype);
    p.out_stride = out_stride_t;
    p.out_stride_s = out_stride_s;
    uint8_t* hq = reinterpret_cast<uint8_t*>(base + ws.hidden);
    CUtensorMap xm, gm, hm, dm;
    rc = encode_rows(&xm, p.xq, n, ex->h, kG8Step);
    if (!rc) rc = encode_rows(&hm, hq, n, ex->i, kG8Step);
    if (!rc)
      rc = encode_weight(&gm, ex->gate_up, ex->h, ex->i, 2, ex->num_experts, ex->gate_up_stride[2],
                         ex->gate_up_stride[1], ex->gate_up_stride[0]);
    if (!rc)
      rc = encode_weight(&dm, ex->down, ex->i, ex->h, 1, ex->num_experts, ex->down_stride[1], 0, ex->down_stride[0]);
    if (rc) return rc;
    F8Args a{};
    a.sorted = reinterpret_cast<int*>(base + ws.sorted);
    a.groups = reinterpret_cast<int4*>(base + ws.groups);
    a.n_groups = reinterpret_cast<int*>(base + ws.n_groups);
    k_fp8_plan<<<kF8PlanCtas, kF8PlanThreads, 2 * sizeof(int) * ex->num_experts, st>>>(
        r, experts_group(ex, n), reinterpret_cast<int*>(base + ws.sorted), reinterpret_cast<int*>(base + ws.place),
        reinterpret_cast<int4*>(base + ws.groups), reinterpret_cast<int*>(base + ws.n_groups));
    rc = check_launch("k_fp8_plan");
    if (rc) return rc;
    rc = launch_rows(p, x_dtype, st);
    if (rc) return rc;
    a.s = s;
    a.err = error_bits;
    a.wait_ns = g_wait_ns;
    a.n = ex->i;
    a.k = ex->h;
    a.sx = p.sx;
    a.scale_rows = n;
    a.ws = ex->gate_up_scale;
    a.hq = hq;
    a.hs = reinterpret_cast<float*>(base + ws.hs);
    rc = launch_grouped<kFp8GateUp>(xm, gm, a, ws.max_groups * fp8_blocks(ex->i), st);
    if (rc) return rc;
    a.n = ex->h;
    a.k = ex->i;
    a.sx = a.hs;
    a.ws = ex->down_scale;
    a.out = out;
    a.out_dtype = out_dtype;
    a.out_stride = out_stride_t;
    a.out_stride_s = out_stride_s;
    a.out_vec = p.out_vec;
    return launch_grouped<kFp8Down>(hm, dm, a, ws.max_groups * ((fp8_blocks(ex->h) + 1) / 2), st);
  }
  StreamArgs a{};
  a.r = r;
  const unsigned groups = static_cast<unsigned>(n);
  const int64_t hs = round_up(ex->i, 4);
  a.x = x;
  a.x_stride = x_stride;
  a.x_vec = rows_vec(x, x_stride, x_dtype);
  a.n = ex->i;
  a.k = ex->h;
  a.w = static_cast<const uint8_t*>(ex->gate_up);
  a.w_stride = ex->gate_up_stride[2];
  a.w_stride_e = ex->gate_up_stride[0];
  a.w_stride_half = ex->gate_up_stride[1];
  a.ws = ex->gate_up_scale;
  a.out = base + ws.hidden;
  a.out_stride = hs;
  rc = launch_stream<kFp8GateUp>(a, x_dtype, groups, false, st);
  if (rc) return rc;
  a.x = base + ws.hidden;
  a.x_stride = hs;
  a.x_vec = 1;
  a.n = ex->h;
  a.k = ex->i;
  a.w = static_cast<const uint8_t*>(ex->down);
  a.w_stride = ex->down_stride[1];
  a.w_stride_e = ex->down_stride[0];
  a.w_stride_half = 0;
  a.ws = ex->down_scale;
  a.out = out;
  a.out_dtype = out_dtype;
  a.out_stride = out_stride_t;
  a.out_stride_s = out_stride_s;
  a.zero_skipped = zero_skipped;
  return launch_stream<kFp8Down>(a, ALUT_F32, groups, true, st);
}

}  // extern "C"
