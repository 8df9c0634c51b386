// C ABI of the 8-bit products (alut_quantize_fp8, alut_linear_fp8, alut_experts_fp8 of
// include/alut.h): argument checks on the host, workspace layout, kernel choice, launches.
#include <algorithm>

#include "alut_fp8.cuh"
#include "alut_host.cuh"

namespace alut {

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
static int launch_stream(const StreamArgs& a, int x_dtype, unsigned groups, bool pdl, cudaStream_t st) {
  const int rows = MODE == kFp8GateUp ? kStreamWRows : 2 * kStreamWRows;
  const dim3 grid(groups, static_cast<unsigned>(ceil_div(a.n, rows)));
  if (grid.y > 65535u) return fail(ALUT_ERANGE, "fp8: %d weight rows", a.n);
  const dim3 block(32 * std::min(kStreamMaxWarps, fp8_blocks(a.k)));
  void (*kern)(StreamArgs) = nullptr;
  if (MODE == kFp8Down || x_dtype == ALUT_F32) kern = k_fp8_stream<float, MODE>;
  if constexpr (MODE != kFp8Down) {
    if (x_dtype == ALUT_BF16) kern = k_fp8_stream<__nv_bfloat16, MODE>;
    if (x_dtype == ALUT_F16) kern = k_fp8_stream<__half, MODE>;
  }
  if (!pdl) {
    kern<<<grid, block, 0, st>>>(a);
    return check_launch("k_fp8_stream");
  }
  const cudaError_t e = launch_pdl(kern, grid, block, 0, st, a);
  if (e != cudaSuccess) return fail(ALUT_ECUDA, "k_fp8_stream: %s", cudaGetErrorString(e));
  return ALUT_OK;
}

// Workspace of alut_experts_fp8, in order; every part starts on 256 bytes.
struct ExpertsWorkspace {
  size_t n_groups, groups, sorted, hidden, total;
  int64_t max_groups;
};
static ExpertsWorkspace experts_layout(const alut_fp8_experts_t* ex, int q, int s) {
  ExpertsWorkspace w{};
  const int64_t n = static_cast<int64_t>(q) * s;
  w.max_groups = ceil_div(n, kStreamRows) + std::min<int64_t>(n, ex->num_experts);
  size_t off = 0;
  w.n_groups = off; off = align256(off + sizeof(int));
  w.groups = off;   off = align256(off + sizeof(int4) * w.max_groups);
  w.sorted = off;   off = align256(off + sizeof(int) * n);
  w.hidden = off;   off = align256(off + sizeof(float) * n * round_up(ex->i, 4));
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
  QuantArgs a{batch, rows, cols, dtype, src, src_stride_b, src_stride, static_cast<uint8_t*>(out), out_stride_b,
              out_stride, scale};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int64_t kb = fp8_blocks(cols);
  if (block_rows == 1) {
    const int64_t n = batch * rows * kb;
    k_fp8_quantize_rows<<<static_cast<unsigned>(std::min<int64_t>((n + 7) / 8, 16 * num_sms())), 256, 0, st>>>(a);
    return check_launch("k_fp8_quantize_rows");
  }
  const int64_t n = batch * ((rows + kFp8Block - 1) / kFp8Block) * kb;
  k_fp8_quantize_blocks<<<static_cast<unsigned>(std::min<int64_t>(n, 1 << 20)), 256, 0, st>>>(a);
  return check_launch("k_fp8_quantize_blocks");
}

size_t alut_linear_fp8_workspace_size(int32_t m, int32_t n, int32_t k) {
  if (m < 0 || n <= 0 || k <= 0) return 0;
  return 256;
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
  if (!workspace || workspace_bytes < need)
    return fail(ALUT_EWORKSPACE, "linear_fp8: workspace has %zu bytes, needs %zu", workspace_bytes, need);
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
  return launch_stream<kFp8Linear>(a, x_dtype, static_cast<unsigned>(ceil_div(m, kStreamRows)), false,
                                   reinterpret_cast<cudaStream_t>(stream));
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
  Fp8Route r{q, s, ex->num_experts, sel, sel_stride, compute, compute_stride, error_bits};
  StreamArgs a{};
  a.r = r;
  const bool planned = n > kStreamMaxSlots;
  unsigned groups = static_cast<unsigned>(n);
  if (planned) {
    a.sorted = reinterpret_cast<int*>(base + ws.sorted);
    a.groups = reinterpret_cast<int4*>(base + ws.groups);
    a.n_groups = reinterpret_cast<int*>(base + ws.n_groups);
    groups = static_cast<unsigned>(ws.max_groups);
    k_fp8_plan<<<1, kFp8PlanThreads, 2 * sizeof(int) * ex->num_experts, st>>>(
        r, kStreamRows, reinterpret_cast<int*>(base + ws.sorted), reinterpret_cast<int4*>(base + ws.groups),
        reinterpret_cast<int*>(base + ws.n_groups));
    rc = check_launch("k_fp8_plan");
    if (rc) return rc;
    if (zero_skipped) {
      k_fp8_zero_skipped<<<std::min(n, 16 * num_sms()), 256, 0, st>>>(r, ex->h, out, out_dtype, out_stride_t,
                                                                     out_stride_s);
      rc = check_launch("k_fp8_zero_skipped");
      if (rc) return rc;
    }
  }
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
  a.zero_skipped = zero_skipped && !planned;
  return launch_stream<kFp8Down>(a, ALUT_F32, groups, true, st);
}

}  // extern "C"
