// extern "C" entry points of the grouped products, the 8-bit integer product and the activation
// checkpoints (declared in include/soap_mi355.h).
#include "products_launch.hpp"

#include "../../include/soap_mi355.h"

namespace soapmi {
// instantiated in the source files of their types
extern template int row_products<ElemF32, KC>(hipStream_t, const RowProblem&, bool);
extern template int row_products<ElemF32, XC>(hipStream_t, const RowProblem&, bool);
extern template int row_products<ElemBF16, KC>(hipStream_t, const RowProblem&, bool);
extern template int row_products<ElemBF16, XC>(hipStream_t, const RowProblem&, bool);
extern template int row_products<ElemF16, KC>(hipStream_t, const RowProblem&, bool);
extern template int row_products<ElemF16, XC>(hipStream_t, const RowProblem&, bool);
extern template int row_products<ElemI8, KC>(hipStream_t, const RowProblem&, bool);
extern template int sum_products<ElemF32>(hipStream_t, const SumProblem&, bool);
extern template int sum_products<ElemBF16>(hipStream_t, const SumProblem&, bool);
extern template int sum_products<ElemF16>(hipStream_t, const SumProblem&, bool);

// The parts' sums, added in order.
static __global__ __launch_bounds__(256) void join_parts_kernel(SumProblem p) {
  const int64_t matrix = (int64_t)p.rows * p.cols, all = matrix * p.groups.experts;
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= all) return;
  float sum = p.partials[at];
  for (int part = 1; part < p.parts; ++part) sum += p.partials[part * all + at];
  const int64_t e = at / matrix, in = at - e * matrix;
  const int64_t r = in / p.cols, c = in - r * p.cols;
  const int64_t to = e * p.stride_d + r * p.ldd + c;
  if (p.out_type == kFloat32) static_cast<float*>(p.d)[to] = sum;
  else if (p.out_type == kBFloat16) static_cast<__bf16*>(p.d)[to] = (__bf16)sum;
  else static_cast<_Float16*>(p.d)[to] = (_Float16)sum;
}

int launch_join(hipStream_t stream, const SumProblem& p) {
  const int64_t all = (int64_t)p.groups.experts * p.rows * p.cols;  // (at most 128 tiles)
  hipLaunchKernelGGL(join_parts_kernel, dim3((unsigned)ceil_div64(all, 256)), dim3(256), 0, stream, p);
  SOAPMI_LAUNCH_CHECK();
  return kOk;
}
}  // namespace soapmi

using namespace soapmi;

namespace {

constexpr int64_t kSizeLimit = (int64_t)1 << 30;

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
int value_bytes(int dtype) { return dtype == kFloat32 ? 4 : 2; }

int check_type(const char* name, int dtype) {
  SOAPMI_REQUIRE(dtype == kFloat32 || dtype == kBFloat16 || dtype == kFloat16,
                 "%s must be 0 (float32), 1 (bfloat16) or 2 (float16), got %d", name, dtype);
  return kOk;
}

int check_sizes(const int64_t* ends, int64_t experts, int64_t tokens, int64_t n, int64_t k) {
  SOAPMI_REQUIRE(experts >= 0 && tokens >= 0 && n >= 0 && k >= 0, "matrix dimensions must be non-negative");
  SOAPMI_REQUIRE(experts < kSizeLimit && tokens < kSizeLimit && n < kSizeLimit && k < kSizeLimit,
                 "matrix dimensions must be below 2^30");
  SOAPMI_REQUIRE(ends || experts <= 1, "ends may be null for a single expert only, got %lld experts", (long long)experts);
  return kOk;
}

// Whether an operand can be fetched straight to LDS: rows that start at multiples of 16 bytes, and offsets
// inside a tile of up to `stored_rows` stored rows that fit the buffer descriptor.
bool direct_ok(const void* base, int64_t ld_bytes, int64_t stored_rows) {
  return aligned16(base) && ld_bytes % 16 == 0 && ld_bytes * stored_rows < kBufferBytes / 2;
}

int check_gradient(int dtype, int out_dtype, const int64_t* ends, int64_t experts, int64_t tokens, int64_t n, int64_t k,
                   int64_t ldg, int64_t ldx, int64_t lddw, int64_t stride_dw) {
  if (int rc = check_type("dtype", dtype)) return rc;
  SOAPMI_REQUIRE(out_dtype == dtype || out_dtype == kFloat32, "out_dtype must be dtype or 0 (float32), got %d", out_dtype);
  if (int rc = check_sizes(ends, experts, tokens, n, k)) return rc;
  SOAPMI_REQUIRE(ldg >= n && ldx >= k && lddw >= k, "leading dimensions are too small");
  SOAPMI_REQUIRE(experts <= 1 || n == 0 || k == 0 || stride_dw >= (n - 1) * lddw + k, "the experts' matrices must not overlap");
  return kOk;
}

// With a workspace for them, long sums for few tiles are cut into parts.
int sum_problem(int dtype, const void* gradient, int64_t ldg, const int64_t* ends, int64_t experts, int64_t tokens, int64_t n,
                int64_t k, int out_dtype, void* dw, int64_t lddw, int64_t stride_dw, void* workspace, size_t workspace_bytes,
                SumProblem* out) {
  SumProblem p = {};
  p.groups = RowGroups{ends, (int)experts, 0, (int)tokens};
  p.r = static_cast<const char*>(gradient);
  p.ldr = ldg * value_bytes(dtype);
  p.rows = (int)n;
  p.cols = (int)k;
  p.d = dw;
  p.ldd = lddw;
  p.stride_d = stride_dw;
  p.out_type = out_dtype;
  p.parts = 1;
  const size_t need = sum_partials_bytes(experts, tokens, n, k);
  if (workspace && need) {
    if (workspace_bytes < need) {
      set_error("workspace holds %zu bytes, %zu are required", workspace_bytes, need);
      return kWorkspaceTooSmall;
    }
    SOAPMI_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 4 == 0, "workspace must be aligned to 4 bytes");
    p.parts = sum_parts(experts, tokens, n, k);
    p.partials = static_cast<float*>(workspace);
  }
  *out = p;
  return kOk;
}

template <class T>
int launch_quantize(hipStream_t stream, const T* x, int64_t ldx, int64_t rows, int64_t cols, int8_t* codes, int64_t ldq,
                    float* scales) {
  const int vec_x = aligned16(x) && ldx * sizeof(T) % 16 == 0;
  const int vec_q = reinterpret_cast<uintptr_t>(codes) % 8 == 0 && ldq % 8 == 0;
  // Long rows take a workgroup each, short ones a wavefront.
  const int64_t grid = cols > 1024 ? rows : ceil_div64(rows, 4);
  SOAPMI_REQUIRE(grid * 256 < (int64_t)1 << 32, "the matrix has too many rows for one launch");
  if (cols > 1024)
    hipLaunchKernelGGL((quantize_rows_kernel<T, 256>), dim3((unsigned)grid), dim3(256), 0, stream, x, ldx, (int)rows,
                       (int)cols, vec_x, codes, ldq, vec_q, scales);
  else
    hipLaunchKernelGGL((quantize_rows_kernel<T, 64>), dim3((unsigned)grid), dim3(256), 0, stream, x, ldx,
                       (int)rows, (int)cols, vec_x, codes, ldq, vec_q, scales);
  SOAPMI_LAUNCH_CHECK();
  return kOk;
}

template <class T>
int launch_checkpoint(hipStream_t stream, const T* x, int64_t ldx, int64_t rows, int64_t cols, int8_t* codes, int64_t ldq,
                      uint8_t* exponents, int64_t lde, int lowest) {
  const int vec_x = aligned16(x) && ldx * sizeof(T) % 16 == 0;
  const int vec_q = reinterpret_cast<uintptr_t>(codes) % 8 == 0 && ldq % 8 == 0;
  const int64_t blocks = ceil_div64(cols, kCheckpointBlock);
  const int64_t grid = ceil_div64(rows * blocks, 16);
  SOAPMI_REQUIRE(grid * 256 < (int64_t)1 << 32, "the matrix has too many blocks for one launch");
  hipLaunchKernelGGL((checkpoint_kernel<T>), dim3((unsigned)grid), dim3(256), 0, stream, x, ldx, rows, (int)cols,
                     (int)blocks, vec_x, codes, ldq, vec_q, exponents, lde, lowest);
  SOAPMI_LAUNCH_CHECK();
  return kOk;
}

template <class T>
int launch_restore(hipStream_t stream, const int8_t* codes, int64_t ldq, const uint8_t* exponents, int64_t lde, int64_t rows,
                   int64_t cols, T* x, int64_t ldx) {
  const int vec_x = aligned16(x) && ldx * sizeof(T) % 16 == 0;
  const int vec_q = reinterpret_cast<uintptr_t>(codes) % 8 == 0 && ldq % 8 == 0;
  const int64_t pieces = ceil_div64(cols, 8);
  const int64_t grid = ceil_div64(rows * pieces, 256);
  SOAPMI_REQUIRE(grid * 256 < (int64_t)1 << 32, "the matrix is too large for one launch");
  hipLaunchKernelGGL((restore_kernel<T>), dim3((unsigned)grid), dim3(256), 0, stream, codes, ldq, vec_q, exponents, lde, rows,
                     (int)cols, (int)pieces, x, ldx, vec_x);
  SOAPMI_LAUNCH_CHECK();
  return kOk;
}

int check_rows(int dtype, const void* x, int64_t ldx, int64_t rows, int64_t cols, const void* codes, int64_t ldq,
               const void* second) {
  if (int rc = check_type("dtype", dtype)) return rc;
  SOAPMI_REQUIRE(rows >= 0 && cols >= 0, "matrix dimensions must be non-negative");
  SOAPMI_REQUIRE(rows < kSizeLimit && cols < kSizeLimit, "matrix dimensions must be below 2^30");
  SOAPMI_REQUIRE(rows == 0 || (cols == 0 ? second != nullptr : x && codes && second), "buffer addresses must be nonzero");
  SOAPMI_REQUIRE(ldx >= cols && ldq >= cols, "leading dimensions are too small");
  return kOk;
}

}  // namespace

extern "C" {

int soapmi_expert_product(int dtype, const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t stride_w,
                          int transposed, const int64_t* ends, int64_t experts, int64_t tokens, int64_t n, int64_t k,
                          int out_dtype, void* y, int64_t ldy, int zero_rest, void* stream) {
  if (int rc = check_type("dtype", dtype)) return rc;
  SOAPMI_REQUIRE(out_dtype == dtype || out_dtype == kFloat32, "out_dtype must be dtype or 0 (float32), got %d", out_dtype);
  if (int rc = check_sizes(ends, experts, tokens, n, k)) return rc;
  const int64_t inner = transposed ? n : k, cols = transposed ? k : n;
  SOAPMI_REQUIRE(ldx >= inner && ldw >= k && ldy >= cols, "leading dimensions are too small");
  SOAPMI_REQUIRE(stride_w >= 0, "stride_w must be non-negative");
  if (tokens == 0 || cols == 0 || (experts == 0 && !zero_rest)) return kOk;
  SOAPMI_REQUIRE(y && (experts == 0 || inner == 0 || (x && w)), "buffer addresses must be nonzero");
  const int size = value_bytes(dtype);
  RowProblem p = {};
  p.groups = RowGroups{ends, (int)experts, zero_rest ? 1 : 0, (int)tokens};
  p.r = static_cast<const char*>(x);
  p.c = static_cast<const char*>(w);
  p.ldr = ldx * size;
  p.ldc = ldw * size;
  p.stride_c = stride_w * size;
  p.cols = (int)cols;
  p.k = (int)inner;
  p.y = y;
  p.ldy = ldy;
  p.out_type = out_dtype;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool direct = direct_ok(x, p.ldr, 256) && direct_ok(w, p.ldc, 256) &&
                      (experts <= 1 || p.stride_c % 16 == 0);
  if (dtype == kFloat32) return transposed ? row_products<ElemF32, XC>(s, p, direct) : row_products<ElemF32, KC>(s, p, direct);
  if (dtype == kBFloat16) return transposed ? row_products<ElemBF16, XC>(s, p, direct) : row_products<ElemBF16, KC>(s, p, direct);
  return transposed ? row_products<ElemF16, XC>(s, p, direct) : row_products<ElemF16, KC>(s, p, direct);
}

int soapmi_expert_weight_gradient(int dtype, const void* gradient, int64_t ldg, const void* x, int64_t ldx,
                                  const int64_t* ends, int64_t experts, int64_t tokens, int64_t n, int64_t k,
                                  int out_dtype, void* dw, int64_t lddw, int64_t stride_dw, void* workspace, size_t workspace_bytes,
                                  void* stream) {
  if (int rc = check_gradient(dtype, out_dtype, ends, experts, tokens, n, k, ldg, ldx, lddw, stride_dw)) return rc;
  if (experts == 0 || n == 0 || k == 0) return kOk;
  SOAPMI_REQUIRE(dw && (tokens == 0 || (gradient && x)), "buffer addresses must be nonzero");
  SumProblem p;
  if (int rc = sum_problem(dtype, gradient, ldg, ends, experts, tokens, n, k, out_dtype, dw, lddw, stride_dw, workspace,
                           workspace_bytes, &p))
    return rc;
  p.c = static_cast<const char*>(x);
  p.ldc = ldx * value_bytes(dtype);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool direct = direct_ok(gradient, p.ldr, 64) && direct_ok(x, p.ldc, 64);
  if (dtype == kFloat32) return sum_products<ElemF32>(s, p, direct);
  return dtype == kBFloat16 ? sum_products<ElemBF16>(s, p, direct) : sum_products<ElemF16>(s, p, direct);
}

size_t soapmi_expert_weight_gradient_workspace_bytes(int64_t experts, int64_t tokens, int64_t n, int64_t k) {
  const bool fits = experts < kSizeLimit && tokens < kSizeLimit && n < kSizeLimit && k < kSizeLimit;  // others are refused
  return fits && experts > 0 && tokens > 0 && n > 0 && k > 0 ? sum_partials_bytes(experts, tokens, n, k) : 0;
}

int soapmi_checkpoint_activations(int dtype, const void* x, int64_t ldx, int64_t rows, int64_t cols, int8_t* codes,
                                  int64_t ldq, uint8_t* exponents, int64_t lde, void* stream) {
  if (int rc = check_rows(dtype, x, ldx, rows, cols, codes, ldq, exponents)) return rc;
  SOAPMI_REQUIRE(lde >= ceil_div64(cols, kCheckpointBlock), "leading dimensions are too small");
  if (rows == 0 || cols == 0) return kOk;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == kFloat32) return launch_checkpoint(s, static_cast<const float*>(x), ldx, rows, cols, codes, ldq, exponents, lde, 1);
  if (dtype == kBFloat16) return launch_checkpoint(s, static_cast<const __bf16*>(x), ldx, rows, cols, codes, ldq, exponents, lde, 1);
  return launch_checkpoint(s, static_cast<const _Float16*>(x), ldx, rows, cols, codes, ldq, exponents, lde, 127 - 24);
}

int soapmi_restore_activations(int dtype, const int8_t* codes, int64_t ldq, const uint8_t* exponents, int64_t lde,
                               int64_t rows, int64_t cols, void* x, int64_t ldx, void* stream) {
  if (int rc = check_rows(dtype, x, ldx, rows, cols, codes, ldq, exponents)) return rc;
  SOAPMI_REQUIRE(lde >= ceil_div64(cols, kCheckpointBlock), "leading dimensions are too small");
  if (rows == 0 || cols == 0) return kOk;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == kFloat32) return launch_restore(s, codes, ldq, exponents, lde, rows, cols, static_cast<float*>(x), ldx);
  if (dtype == kBFloat16) return launch_restore(s, codes, ldq, exponents, lde, rows, cols, static_cast<__bf16*>(x), ldx);
  return launch_restore(s, codes, ldq, exponents, lde, rows, cols, static_cast<_Float16*>(x), ldx);
}

int soapmi_quantize_rows(int dtype, const void* x, int64_t ldx, int64_t rows, int64_t cols, int8_t* codes, int64_t ldq,
                         float* scales, void* stream) {
  if (int rc = check_rows(dtype, x, ldx, rows, cols, codes, ldq, scales)) return rc;
  if (rows == 0) return kOk;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == kFloat32) return launch_quantize(s, static_cast<const float*>(x), ldx, rows, cols, codes, ldq, scales);
  if (dtype == kBFloat16) return launch_quantize(s, static_cast<const __bf16*>(x), ldx, rows, cols, codes, ldq, scales);
  return launch_quantize(s, static_cast<const _Float16*>(x), ldx, rows, cols, codes, ldq, scales);
}

int soapmi_int8_product(const int8_t* codes, int64_t ldq, const float* scales, const int8_t* w_codes, int64_t ldw,
                        const float* w_scales, int64_t tokens, int64_t n, int64_t k, int out_dtype, void* y, int64_t ldy,
                        void* stream) {
  if (int rc = check_type("out_dtype", out_dtype)) return rc;
  if (int rc = check_sizes(nullptr, 1, tokens, n, k)) return rc;
  SOAPMI_REQUIRE(k <= 131071, "k must be at most 131071: the integer sums would leave 32 bits");
  SOAPMI_REQUIRE(ldq >= k && ldw >= k && ldy >= n, "leading dimensions are too small");
  if (tokens == 0 || n == 0) return kOk;
  SOAPMI_REQUIRE(y && scales && w_scales && (k == 0 || (codes && w_codes)), "buffer addresses must be nonzero");
  RowProblem p = {};
  p.groups = RowGroups{nullptr, 1, 0, (int)tokens};
  p.r = reinterpret_cast<const char*>(codes);
  p.c = reinterpret_cast<const char*>(w_codes);
  p.ldr = ldq;
  p.ldc = ldw;
  p.cols = (int)n;
  p.k = (int)k;
  p.y = y;
  p.ldy = ldy;
  p.out_type = out_dtype;
  p.token_scale = scales;
  p.channel_scale = w_scales;
  const bool direct = direct_ok(codes, ldq, 256) && direct_ok(w_codes, ldw, 256);
  return row_products<ElemI8, KC>(static_cast<hipStream_t>(stream), p, direct);
}

}  // extern "C"
