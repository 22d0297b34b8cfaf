// C-ABI entry points of libflash_hypercons_hip.so (declared in
// include/flash_hypercons.h): argument validation, operand description and
// kernel selection.  Replaces the reference's host launcher
// csrc/matrix_exp.cu:13-86 without its FP32/contiguous/padded staging copies:
// the kernels read the caller's strided storage directly and write only the
// logical n x n block.
#include <cmath>
#include <string>

#include "fh_kernels.h"
#include "fh_plan.h"
#include "fh_rows.h"
#include "flash_hypercons.h"

namespace {

thread_local std::string g_error;

// The reference's input check message (csrc/matrix_exp.cu:52-55).
constexpr const char* kInputMessage =
    "expected a strided CUDA [B, N, N] tensor, 2 <= N <= 32, in float32, float16, or bfloat16";
constexpr const char* kDirectionMessage = "matrix exponential direction must match the input";

int fail(int code, const std::string& message) {
  g_error = message;
  return code;
}

int element_size(int dtype) { return dtype == FH_DTYPE_F32 ? 4 : 2; }

bool aligned(const void* p, int64_t bytes) {
  return (reinterpret_cast<uintptr_t>(p) % static_cast<uintptr_t>(bytes)) == 0;
}

fh::Operand make_operand(const void* data, const int64_t strides[3], int neg, int dtype, int n) {
  fh::Operand op;
  op.data = data;
  op.sb = strides[0];
  op.sr = strides[1];
  op.sc = strides[2];
  op.sign = neg ? -1.f : 1.f;
  op.vec = fh::kVecNone;
  op.dense = 0;
  if (n == 4 || n == 8) {
    // Every row (or column) of the matrix is made of aligned 4-element
    // vectors when its elements are adjacent and every matrix/row (column)
    // start keeps the vector alignment; consecutive matrices are one
    // contiguous block (`dense`) when they are packed as well.
    const int64_t vbytes = 4 * element_size(dtype);
    const bool base_ok = aligned(data, vbytes) && strides[0] % 4 == 0;
    const bool packed = strides[0] == n * n && aligned(data, 16);
    if (base_ok && strides[2] == 1 && strides[1] % 4 == 0) {
      op.vec = fh::kVecRows;
      op.dense = packed && strides[1] == n;
    } else if (base_ok && strides[1] == 1 && strides[2] % 4 == 0) {
      op.vec = fh::kVecCols;
      op.dense = packed && strides[2] == n;
    }
  }
  return op;
}

// The P = 16/32 kernels address one matrix through a buffer resource with
// 32-bit offsets: its footprint ((n - 1) * (sr + sc) + 1 elements) must stay
// below 2 GiB and its strides non-negative.  Other operands go to the
// one-wavefront-per-matrix kernel, which indexes in 64 bits.
bool tile_addressable(const fh::Operand& op, int n, int dtype) {
  if (op.sr < 0 || op.sc < 0 || op.sb < 0) return false;
  const int64_t limit = (int64_t{1} << 31) - 1;
  const int64_t es = element_size(dtype);
  if (op.sr > limit || op.sc > limit) return false;
  return ((n - 1) * (op.sr + op.sc) + 1) * es <= limit;
}

int validate(const void* input, const int64_t* strides, int dtype, int64_t batch, int n, const void* out) {
  if (n < 2 || n > 32 || (dtype != FH_DTYPE_F32 && dtype != FH_DTYPE_BF16 && dtype != FH_DTYPE_F16) || batch < 0)
    return fail(FH_ERR_INVALID_ARGUMENT, kInputMessage);
  if (batch > 0 && (input == nullptr || strides == nullptr || out == nullptr))
    return fail(FH_ERR_INVALID_ARGUMENT, "null input, stride or output pointer");
  return FH_OK;
}

int launch(const void* input, const int64_t input_strides[3], int input_neg, const void* direction,
           const int64_t direction_strides[3], int direction_neg, void* out, int dtype, int64_t batch, int n,
           int variant, int32_t* s_out, hipStream_t stream) {
  int rc = validate(input, input_strides, dtype, batch, n, out);
  if (rc != FH_OK) return rc;
  if (variant != FH_VARIANT_AUTO && variant != FH_VARIANT_GENERIC)
    return fail(FH_ERR_INVALID_ARGUMENT, "unknown kernel variant");
  const bool pair = direction != nullptr;
  if (pair && batch > 0 && direction_strides == nullptr) return fail(FH_ERR_INVALID_ARGUMENT, kDirectionMessage);
  if (batch == 0) return FH_OK;  // csrc/matrix_exp.cu:62-64
  fh::ExpmArgs args;
  args.x = make_operand(input, input_strides, input_neg, dtype, n);
  if (pair) {
    args.g = make_operand(direction, direction_strides, direction_neg, dtype, n);
  } else {
    args.g = args.x;
  }
  args.out = out;
  args.s_out = s_out;
  args.batch = batch;
  args.n = n;
  const int P = n <= 4 ? 4 : n <= 8 ? 8 : n <= 16 ? 16 : 32;  // csrc/matrix_exp.cu:65
  hipError_t err;
  if (variant == FH_VARIANT_GENERIC) {
    err = fh::launch_generic(args, dtype, P, pair, stream);
  } else if (P == 4) {
    err = fh::launch_p4(args, dtype, pair, stream);
  } else if (P == 8) {
    err = fh::launch_oct(args, dtype, pair, stream);
  } else if (tile_addressable(args.x, n, dtype) && (!pair || tile_addressable(args.g, n, dtype))) {
    err = fh::launch_tile(args, dtype, P, pair, stream);
  } else {
    err = fh::launch_generic(args, dtype, P, pair, stream);
  }
  if (err != hipSuccess) return fail(FH_ERR_LAUNCH, std::string("kernel launch failed: ") + hipGetErrorString(err));
  g_error.clear();
  return FH_OK;
}

// Operands of the fused stream mixing: H any strides; X (and dY) [B, n, C]
// with contiguous, 16-byte aligned rows of a whole number of 16-byte vectors,
// each token's rows spanning less than 2 GiB.
// Rows of a streamed operand ([B, n, C], unit column stride): 16-byte aligned,
// strides and C whole 16-byte vectors, each token's rows spanning < 2 GiB.
constexpr int64_t kSpan = int64_t{1} << 31;  // bytes one token's rows may span (32-bit buffer offsets)

// Layout the streaming kernels read in place: contiguous, 16-byte aligned rows
// whose length and strides are whole 16-byte vectors.
bool stream_rows_ok(const void* p, const int64_t* st, int64_t cols, int dtype) {
  const int64_t v = 16 / element_size(dtype);
  return st != nullptr && aligned(p, 16) && st[2] == 1 && st[0] >= 0 && st[1] >= 0 && st[0] % v == 0 &&
         st[1] % v == 0 && cols % v == 0;
}

// The same with dwords for vectors: what the fused kernels' ragged variants read.
bool dword_rows_ok(const void* p, const int64_t* st, int64_t cols, int dtype) {
  const int64_t v = 4 / element_size(dtype);
  return st != nullptr && aligned(p, 4) && st[2] == 1 && st[0] >= 0 && st[1] >= 0 && st[0] % v == 0 &&
         st[1] % v == 0 && cols % v == 0;
}

// One token's n rows, read through row stride st[1], and the contiguous output
// token (n * cols elements) each span < 2 GiB: the kernels address a token
// through one buffer resource with 32-bit offsets.
bool stream_span_ok(const int64_t* st, int n, int64_t cols, int dtype) {
  const int64_t es = element_size(dtype);
  return st[1] < kSpan && cols < kSpan && ((n - 1) * st[1] + cols) * es < kSpan && n * cols * es < kSpan;
}

std::string span_message(const char* op) {
  return std::string(op) + ": one token's rows of X, dY and of the output must each span less than 2 GiB";
}

bool known_dtype(int dtype) { return dtype == FH_DTYPE_F32 || dtype == FH_DTYPE_BF16 || dtype == FH_DTYPE_F16; }

std::string rows_message(const char* op, int dtype) {
  return std::string(op) + ": X and dY need contiguous, 16-byte aligned rows whose length C and strides are multiples of " +
         std::to_string(16 / element_size(dtype)) + " elements";
}

int validate_hc(const void* h, const int64_t* hs, const void* x, const int64_t* xs, const void* g, const int64_t* gs,
                const void* out, int dtype, int64_t batch, int n, int64_t cols) {
  if (n < 2 || n > 4 || !known_dtype(dtype) || batch < 0 || cols < 1)
    return fail(FH_ERR_INVALID_ARGUMENT,
                "hc_mix: expected H [B, n, n] and X [B, n, C] with 2 <= n <= 4, C >= 1, in float32, float16, or "
                "bfloat16");
  if (batch == 0) return FH_OK;
  if (h == nullptr || hs == nullptr || x == nullptr || xs == nullptr || out == nullptr)
    return fail(FH_ERR_INVALID_ARGUMENT, "hc_mix: null pointer");
  if (!stream_rows_ok(x, xs, cols, dtype) || (g != nullptr && !stream_rows_ok(g, gs, cols, dtype)) ||
      !aligned(out, 16))
    return fail(FH_ERR_INVALID_ARGUMENT, rows_message("hc_mix", dtype));
  if (!stream_span_ok(xs, n, cols, dtype) || (g != nullptr && !stream_span_ok(gs, n, cols, dtype)))
    return fail(FH_ERR_INVALID_ARGUMENT, span_message("hc_mix"));
  return FH_OK;
}

// The apply entry points (5 <= n <= 8): E is FP32 [batch, n, n], contiguous.
int validate_apply(const float* e, const void* x, const int64_t* xs, const void* g, const int64_t* gs,
                   const void* out, int dtype, int64_t batch, int n, int64_t cols) {
  if (n < 5 || n > 8 || !known_dtype(dtype) || batch < 0 || cols < 1)
    return fail(FH_ERR_INVALID_ARGUMENT,
                "hc_apply: expected E [B, n, n] (float32) and X [B, n, C] with 5 <= n <= 8, C >= 1, in float32, "
                "float16, or bfloat16");
  if (batch == 0) return FH_OK;
  if (e == nullptr || x == nullptr || xs == nullptr || out == nullptr)
    return fail(FH_ERR_INVALID_ARGUMENT, "hc_apply: null pointer");
  if (!aligned(e, 4)) return fail(FH_ERR_INVALID_ARGUMENT, "hc_apply: E must be 4-byte aligned float32");
  if (!stream_rows_ok(x, xs, cols, dtype) || (g != nullptr && !stream_rows_ok(g, gs, cols, dtype)) ||
      !aligned(out, 16))
    return fail(FH_ERR_INVALID_ARGUMENT, rows_message("hc_apply", dtype));
  if (!stream_span_ok(xs, n, cols, dtype) || (g != nullptr && !stream_span_ok(gs, n, cols, dtype)))
    return fail(FH_ERR_INVALID_ARGUMENT, span_message("hc_apply"));
  return FH_OK;
}

// ---- layer norm, linear, clipping ------------------------------------------------

int launched(hipError_t err) {
  if (err != hipSuccess) return fail(FH_ERR_LAUNCH, std::string("kernel launch failed: ") + hipGetErrorString(err));
  g_error.clear();
  return FH_OK;
}

// The workspace protocol of calls that need `need` bytes: FH_OK to go on, with
// `*query` set where only the size was asked for.
int check_workspace(const char* op, void* workspace, int64_t* bytes, int64_t need, bool* query) {
  if (bytes == nullptr) return fail(FH_ERR_INVALID_ARGUMENT, std::string(op) + ": null workspace size");
  *query = workspace == nullptr;
  if (*query) {
    *bytes = need;
    g_error.clear();
    return FH_OK;
  }
  if (*bytes < need || (need > 0 && !aligned(workspace, 16)))
    return fail(FH_ERR_INVALID_ARGUMENT, std::string(op) + ": the workspace needs " + std::to_string(need) +
                                             " bytes, 16-byte aligned");
  return FH_OK;
}

bool rows_ok(const void* p, int64_t stride, int dtype) { return p != nullptr && stride >= 0 && aligned(p, element_size(dtype)); }

int validate_norm(const void* x, int64_t x_stride, const void* y, int param_dtype, int dtype, int64_t rows,
                  int64_t cols) {
  if (!known_dtype(dtype) || (param_dtype != dtype && param_dtype != FH_DTYPE_F32) || rows < 0 ||
      rows >= (int64_t{1} << 31) || cols < 1 || cols >= (int64_t{1} << 30))
    return fail(FH_ERR_INVALID_ARGUMENT,
                "layer_norm: expected x [rows, cols] in float32, float16, or bfloat16 with fewer than 2^31 rows and "
                "1 <= cols < 2^30, and weight and bias of its type or float32");
  if (rows > 0 && (!rows_ok(x, x_stride, dtype) || !rows_ok(y, 0, dtype)))
    return fail(FH_ERR_INVALID_ARGUMENT, "layer_norm: null or misaligned pointer, or negative stride");
  return FH_OK;
}

int validate_linear(const fh::LinearArgs& a) {
  constexpr int64_t most = int64_t{1} << 22;
  if (!known_dtype(a.dtype) || (a.bias_dtype != a.dtype && a.bias_dtype != FH_DTYPE_F32) || a.rows < 0 ||
      a.rows >= (int64_t{1} << 30) || a.cols < 1 || a.cols >= most || a.outs < 1 || a.outs >= most)
    return fail(FH_ERR_INVALID_ARGUMENT,
                "linear: expected x [rows, cols] and weight [outs, cols] in float32, float16, or bfloat16 with fewer "
                "than 2^30 rows and 1 <= cols, outs < 2^22, and a bias of their type or float32");
  if (a.act < FH_ACT_NONE || a.act > FH_ACT_SILU) return fail(FH_ERR_INVALID_ARGUMENT, "linear: unknown activation");
  return FH_OK;
}

int validate_clip(const char* op, int count, const void* const* grads, void* const* out, const int64_t* sizes,
                  const int* dtypes, double norm_type, const float* norm, int* power) {
  if (norm_type != 1.0 && norm_type != 2.0 && !(std::isinf(norm_type) && norm_type > 0))
    return fail(FH_ERR_INVALID_ARGUMENT, std::string(op) + ": norm_type is 1, 2 or infinity");
  *power = std::isinf(norm_type) ? 0 : static_cast<int>(norm_type);
  if (count < 0 || norm == nullptr || (count > 0 && (grads == nullptr || sizes == nullptr || dtypes == nullptr)))
    return fail(FH_ERR_INVALID_ARGUMENT, std::string(op) + ": null list or negative count");
  for (int i = 0; i < count; ++i) {
    if (sizes[i] < 0 || !known_dtype(dtypes[i]))
      return fail(FH_ERR_INVALID_ARGUMENT, std::string(op) + ": expected float32, float16, or bfloat16 arrays");
    if (sizes[i] > 0 && (!rows_ok(grads[i], 0, dtypes[i]) || (out != nullptr && !rows_ok(out[i], 0, dtypes[i]))))
      return fail(FH_ERR_INVALID_ARGUMENT, std::string(op) + ": null or misaligned array");
  }
  return FH_OK;
}

}  // namespace

namespace fh {

Operand hc_operand(const void* h, const int64_t strides[3], int neg, int dtype) {
  return make_operand(h, strides, neg, dtype, 0);
}

int64_t compute_units() {
  static PerDevice units;
  int device = 0;
  if (hipGetDevice(&device) != hipSuccess) return 1;
  return units.get(device, [device] {
    int cus = 0;
    return hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, device) == hipSuccess ? cus : 0;
  });
}

int64_t resident_blocks(const void* kernel, int block) {
  int per_cu = 0;
  if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&per_cu, kernel, block, 0) != hipSuccess) per_cu = 1;
  return (per_cu > 0 ? per_cu : 1) * compute_units();
}

}  // namespace fh

extern "C" {

int fh_matrix_exp(const void* input, const int64_t strides[3], int input_neg, void* out, int dtype, int64_t batch,
                  int n, hipStream_t stream) {
  return launch(input, strides, input_neg, nullptr, nullptr, 0, out, dtype, batch, n, FH_VARIANT_AUTO, nullptr,
                stream);
}

int fh_frechet(const void* input, const int64_t input_strides[3], int input_neg, const void* direction,
               const int64_t direction_strides[3], int direction_neg, void* out, int dtype, int64_t batch, int n,
               hipStream_t stream) {
  if (batch > 0 && direction == nullptr) return fail(FH_ERR_INVALID_ARGUMENT, kDirectionMessage);
  return launch(input, input_strides, input_neg, direction, direction_strides, direction_neg, out, dtype, batch, n,
                FH_VARIANT_AUTO, nullptr, stream);
}

int fh_expm_launch(const void* input, const int64_t input_strides[3], int input_neg, const void* direction,
                   const int64_t direction_strides[3], int direction_neg, void* out, int dtype, int64_t batch, int n,
                   int variant, int32_t* s_out, hipStream_t stream) {
  return launch(input, input_strides, input_neg, direction, direction_strides, direction_neg, out, dtype, batch, n,
                variant, s_out, stream);
}

int fh_expm_params(const void* input, const int64_t input_strides[3], int input_neg, const void* direction,
                   const int64_t direction_strides[3], int direction_neg, int dtype, int64_t batch, int n,
                   int32_t* params, double* norms, hipStream_t stream) {
  int rc = validate(input, input_strides, dtype, batch, n, params);
  if (rc != FH_OK) return rc;
  const bool pair = direction != nullptr;
  if (pair && batch > 0 && direction_strides == nullptr) return fail(FH_ERR_INVALID_ARGUMENT, kDirectionMessage);
  if (batch == 0) return FH_OK;
  fh::ExpmArgs args;
  args.x = make_operand(input, input_strides, input_neg, dtype, n);
  args.g = pair ? make_operand(direction, direction_strides, direction_neg, dtype, n) : args.x;
  args.out = nullptr;
  args.s_out = nullptr;
  args.batch = batch;
  args.n = n;
  const hipError_t err = fh::launch_params(args, dtype, pair, params, norms, stream);
  if (err != hipSuccess) return fail(FH_ERR_LAUNCH, std::string("kernel launch failed: ") + hipGetErrorString(err));
  g_error.clear();
  return FH_OK;
}

int fh_hc_mix(const void* h, const int64_t h_strides[3], int h_neg, const void* x, const int64_t x_strides[3],
              void* y, float* e_out, int dtype, int64_t batch, int n, int64_t cols, hipStream_t stream) {
  int rc = validate_hc(h, h_strides, x, x_strides, nullptr, nullptr, y, dtype, batch, n, cols);
  if (rc != FH_OK || batch == 0) return rc;
  const hipError_t err = fh::launch_hc_mix(fh::hc_operand(h, h_strides, h_neg, dtype), x, x_strides, nullptr,
                                           nullptr, y, nullptr, e_out, dtype, batch, n, cols, stream);
  if (err != hipSuccess) return fail(FH_ERR_LAUNCH, std::string("kernel launch failed: ") + hipGetErrorString(err));
  g_error.clear();
  return FH_OK;
}

int fh_hc_mix_backward(const void* h, const int64_t h_strides[3], int h_neg, const void* x,
                       const int64_t x_strides[3], const void* grad, const int64_t grad_strides[3], void* dh,
                       void* dx, float* de_out, int dtype, int64_t batch, int n, int64_t cols, hipStream_t stream) {
  int rc = validate_hc(h, h_strides, x, x_strides, grad, grad_strides, dx, dtype, batch, n, cols);
  if (rc != FH_OK) return rc;
  if (batch > 0 && (grad == nullptr || dh == nullptr))
    return fail(FH_ERR_INVALID_ARGUMENT, "hc_mix: null grad or dh pointer");
  if (batch == 0) return FH_OK;
  const hipError_t err = fh::launch_hc_mix(fh::hc_operand(h, h_strides, h_neg, dtype), x, x_strides, grad,
                                           grad_strides, dx, dh, de_out, dtype, batch, n, cols, stream);
  if (err != hipSuccess) return fail(FH_ERR_LAUNCH, std::string("kernel launch failed: ") + hipGetErrorString(err));
  g_error.clear();
  return FH_OK;
}

int fh_hc_mix_dwords(const void* h, const int64_t h_strides[3], int h_neg, const void* x, const int64_t x_strides[3],
                     const void* grad, const int64_t* grad_strides, void* dh, void* out, float* aux, int dtype,
                     int64_t batch, int n, int64_t cols, hipStream_t stream) {
  if (n < 2 || n > 4 || !known_dtype(dtype) || batch < 0 || cols < 1)
    return fail(FH_ERR_INVALID_ARGUMENT,
                "hc_mix: expected H [B, n, n] and X [B, n, C] with 2 <= n <= 4, C >= 1, in float32, float16, or "
                "bfloat16");
  if (batch == 0) return FH_OK;
  if (h == nullptr || h_strides == nullptr || x == nullptr || x_strides == nullptr || out == nullptr ||
      (grad != nullptr && (grad_strides == nullptr || dh == nullptr)))
    return fail(FH_ERR_INVALID_ARGUMENT, "hc_mix: null pointer");
  if (!dword_rows_ok(x, x_strides, cols, dtype) || (grad != nullptr && !dword_rows_ok(grad, grad_strides, cols, dtype)) ||
      !aligned(out, 4))
    return fail(FH_ERR_INVALID_ARGUMENT, "hc_mix: X and dY need contiguous, 4-byte aligned rows of whole dwords");
  // The span of the rows padded to whole vectors: the limit of the padded layout.
  const int64_t v = 16 / element_size(dtype);
  const int64_t padded = cols < kSpan ? (cols + v - 1) / v * v : cols;
  if (!stream_span_ok(x_strides, n, padded, dtype) ||
      (grad != nullptr && !stream_span_ok(grad_strides, n, padded, dtype)))
    return fail(FH_ERR_INVALID_ARGUMENT, span_message("hc_mix"));
  const hipError_t err = fh::launch_hc_mix(fh::hc_operand(h, h_strides, h_neg, dtype), x, x_strides, grad,
                                           grad_strides, out, dh, aux, dtype, batch, n, cols, stream);
  if (err != hipSuccess) return fail(FH_ERR_LAUNCH, std::string("kernel launch failed: ") + hipGetErrorString(err));
  g_error.clear();
  return FH_OK;
}

int fh_hc_apply(const float* e, const void* x, const int64_t x_strides[3], void* y, int dtype, int64_t batch, int n,
                int64_t cols, hipStream_t stream) {
  g_error.clear();
  const int rc = validate_apply(e, x, x_strides, nullptr, nullptr, y, dtype, batch, n, cols);
  if (rc != FH_OK || batch == 0) return rc;
  const hipError_t err =
      fh::launch_hc_apply(e, x, x_strides, nullptr, nullptr, y, nullptr, dtype, batch, n, cols, stream);
  if (err != hipSuccess) return fail(FH_ERR_LAUNCH, std::string("kernel launch failed: ") + hipGetErrorString(err));
  return FH_OK;
}

int fh_hc_apply_backward(const float* e, const void* x, const int64_t x_strides[3], const void* grad,
                         const int64_t grad_strides[3], void* dx, float* de, int dtype, int64_t batch, int n,
                         int64_t cols, hipStream_t stream) {
  g_error.clear();
  const int rc = validate_apply(e, x, x_strides, grad, grad_strides, dx, dtype, batch, n, cols);
  if (rc != FH_OK) return rc;
  if (batch > 0 && (grad == nullptr || de == nullptr))
    return fail(FH_ERR_INVALID_ARGUMENT, "hc_apply: null grad or de pointer");
  if (batch > 0 && !aligned(de, 4)) return fail(FH_ERR_INVALID_ARGUMENT, "hc_apply: dE must be 4-byte aligned float32");
  if (batch == 0) return FH_OK;
  const hipError_t err = fh::launch_hc_apply(e, x, x_strides, grad, grad_strides, dx, de, dtype, batch, n, cols, stream);
  if (err != hipSuccess) return fail(FH_ERR_LAUNCH, std::string("kernel launch failed: ") + hipGetErrorString(err));
  return FH_OK;
}

int fh_layer_norm(const void* x, int64_t x_stride, const void* weight, const void* bias, int param_dtype, double eps,
                  void* y, float* stats, int dtype, int64_t rows, int64_t cols, hipStream_t stream) {
  const int rc = validate_norm(x, x_stride, y, param_dtype, dtype, rows, cols);
  if (rc != FH_OK) return rc;
  if (rows == 0) return launched(hipSuccess);
  fh::NormArgs a{};
  a.x = x;
  a.x_stride = x_stride;
  a.weight = weight;
  a.bias = bias;
  a.params_f32 = param_dtype == FH_DTYPE_F32;
  a.eps = static_cast<float>(eps);
  a.y = y;
  a.stats = stats;
  a.rows = rows;
  a.cols = cols;
  return launched(fh::launch_norm(a, dtype, stream));
}

int fh_layer_norm_backward(const void* x, int64_t x_stride, const void* grad, int64_t grad_stride, const void* weight,
                           int param_dtype, const float* stats, void* dx, void* dweight, void* dbias, void* workspace,
                           int64_t* workspace_bytes, int dtype, int64_t rows, int64_t cols, hipStream_t stream) {
  int rc = validate_norm(x, x_stride, dx, param_dtype, dtype, rows, cols);
  if (rc != FH_OK) return rc;
  if (rows == 0) return fail(FH_ERR_INVALID_ARGUMENT, "layer_norm: no rows, whose gradients are zeros of the caller's");
  if (!rows_ok(grad, grad_stride, dtype) || stats == nullptr)
    return fail(FH_ERR_INVALID_ARGUMENT, "layer_norm: null or misaligned pointer, or negative stride");
  const bool params = dweight != nullptr || dbias != nullptr;
  const int64_t need = params ? fh::norm_blocks(dtype, rows, cols) * 2 * cols * static_cast<int64_t>(sizeof(float)) : 0;
  bool query = false;
  rc = check_workspace("layer_norm", workspace, workspace_bytes, need, &query);
  if (rc != FH_OK || query) return rc;
  fh::NormArgs a{};
  a.x = x;
  a.x_stride = x_stride;
  a.grad = grad;
  a.grad_stride = grad_stride;
  a.weight = weight;
  a.params_f32 = param_dtype == FH_DTYPE_F32;
  a.y = dx;
  a.stats = const_cast<float*>(stats);
  a.partial = params ? static_cast<float*>(workspace) : nullptr;
  a.rows = rows;
  a.cols = cols;
  return launched(fh::launch_norm_backward(a, dweight, dbias, param_dtype, dtype, stream));
}

int fh_linear(const void* x, int64_t x_stride, const void* weight, int64_t weight_stride, const void* bias,
              int bias_dtype, const void* residual, int64_t residual_stride, int activation, void* y, void* saved,
              void* workspace, int64_t* workspace_bytes, int dtype, int64_t rows, int64_t cols, int64_t outs,
              hipStream_t stream) {
  fh::LinearArgs a{};
  a.x = x;
  a.x_stride = x_stride;
  a.weight = weight;
  a.w_stride = weight_stride;
  a.bias = bias;
  a.bias_dtype = bias_dtype;
  a.residual = residual;
  a.r_stride = residual_stride;
  a.act = activation;
  a.dtype = dtype;
  a.saved = saved;
  a.y = y;
  a.rows = rows;
  a.cols = cols;
  a.outs = outs;
  int rc = validate_linear(a);
  if (rc != FH_OK) return rc;
  int64_t need = 0;
  bool query = false;
  if (rows > 0) {
    if (!rows_ok(x, x_stride, dtype) || !rows_ok(weight, weight_stride, dtype) || !rows_ok(y, 0, dtype) ||
        (residual != nullptr && !rows_ok(residual, residual_stride, dtype)) ||
        (bias != nullptr && !aligned(bias, element_size(bias_dtype))))
      return fail(FH_ERR_INVALID_ARGUMENT, "linear: null or misaligned pointer, or negative stride");
    (void)fh::launch_linear(a, nullptr, &need, stream);
  }
  rc = check_workspace("linear", workspace, workspace_bytes, need, &query);
  if (rc != FH_OK || query) return rc;
  return launched(rows > 0 ? fh::launch_linear(a, workspace, nullptr, stream) : hipSuccess);
}

int fh_linear_backward(const void* x, int64_t x_stride, const void* weight, int64_t weight_stride, const void* grad,
                       int64_t grad_stride, const void* saved, int activation, void* dx, void* dweight, void* dbias,
                       int bias_dtype, void* workspace, int64_t* workspace_bytes, int dtype, int64_t rows,
                       int64_t cols, int64_t outs, hipStream_t stream) {
  fh::LinearArgs a{};
  a.x = x;
  a.x_stride = x_stride;
  a.weight = weight;
  a.w_stride = weight_stride;
  a.grad = grad;
  a.g_stride = grad_stride;
  a.bias_dtype = bias_dtype;
  a.act = activation;
  a.dtype = dtype;
  a.saved = const_cast<void*>(saved);
  a.dx = dx;
  a.dweight = dweight;
  a.dbias = dbias;
  a.rows = rows;
  a.cols = cols;
  a.outs = outs;
  int rc = validate_linear(a);
  if (rc != FH_OK) return rc;
  if (rows == 0) return fail(FH_ERR_INVALID_ARGUMENT, "linear: no rows, whose gradients are zeros of the caller's");
  if ((activation != FH_ACT_NONE) != (saved != nullptr))
    return fail(FH_ERR_INVALID_ARGUMENT, "linear: the backward takes the forward's `saved` with an activation only");
  if (!rows_ok(grad, grad_stride, dtype) || (dweight != nullptr && !rows_ok(x, x_stride, dtype)) ||
      (dx != nullptr && !rows_ok(weight, weight_stride, dtype)))
    return fail(FH_ERR_INVALID_ARGUMENT, "linear: null or misaligned pointer, or negative stride");
  int64_t need = 0;
  bool query = false;
  (void)fh::launch_linear_backward(a, nullptr, &need, stream);
  rc = check_workspace("linear", workspace, workspace_bytes, need, &query);
  if (rc != FH_OK || query) return rc;
  return launched(fh::launch_linear_backward(a, workspace, nullptr, stream));
}

int fh_grad_norm(int count, const void* const* grads, const int64_t* sizes, const int* dtypes, double norm_type,
                 float* norm, void* workspace, int64_t* workspace_bytes, hipStream_t stream) {
  int power = 0;
  int rc = validate_clip("grad_norm", count, grads, nullptr, sizes, dtypes, norm_type, norm, &power);
  if (rc != FH_OK) return rc;
  const fh::ClipList list{count, grads, nullptr, sizes, dtypes};
  bool query = false;
  rc = check_workspace("grad_norm", workspace, workspace_bytes, fh::clip_partials(list) * 8, &query);
  if (rc != FH_OK || query) return rc;
  return launched(fh::launch_clip(list, power, 0.0, false, norm, static_cast<double*>(workspace), stream));
}

int fh_clip_gradients(int count, const void* const* grads, void* const* out, const int64_t* sizes, const int* dtypes,
                      double norm_type, double max_norm, float* norm, void* workspace, int64_t* workspace_bytes,
                      hipStream_t stream) {
  int power = 0;
  int rc = validate_clip("clip_gradients", count, grads, out, sizes, dtypes, norm_type, norm, &power);
  if (rc != FH_OK) return rc;
  const fh::ClipList list{count, grads, out, sizes, dtypes};
  bool query = false;
  rc = check_workspace("clip_gradients", workspace, workspace_bytes, fh::clip_partials(list) * 8, &query);
  if (rc != FH_OK || query) return rc;
  return launched(fh::launch_clip(list, power, max_norm, true, norm, static_cast<double*>(workspace), stream));
}

const char* fh_last_error(void) { return g_error.c_str(); }

const char* fh_version(void) { return "0.1.0"; }

}  // extern "C"
