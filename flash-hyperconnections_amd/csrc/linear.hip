// The linear layer around its matrix products:
//   z = x W^T + b,  y = act(z) + residual;
//   dz = g act'(z),  dx = dz W,  dW = dz^T x,  db = sum over rows of dz.
//
// The products take 16-bit operands whose rows are 16-byte aligned and whole 16-byte
// vectors; others are laid out anew first, in padded rows (prepare_kernel).  FP32
// operands they take as they are.
//
// dz is formed by the same kernel, together with the column sums that make db.  It is
// rounded to the storage type, as operands of 16-bit products have to be; db adds the
// values before that rounding.  With an activation this doubles the variance of dx's and
// dW's errors: 0.0024 of their size in bf16 and 0.0003 in FP16 (root mean square, against 64
// bits, gelu and normal operands), where the results' own rounding makes 0.0017 and 0.0002.
// Without one dz is the upstream gradient itself and loses nothing.
#include <algorithm>

#include "fh_plan.h"
#include "linear.h"

namespace fh {
namespace {

struct PrepareArgs {
  const void* src;   // [rows, cols], rows src_stride elements apart
  int64_t src_stride;
  const void* saved; // with an activation: [rows, cols] contiguous
  int act;
  void* out;         // [rows, ld], zero past cols; or null
  int64_t ld;
  float* partial;    // [gridDim.y, cols] column sums, or null
  int64_t rows;
  int cols;
};

// Four wavefronts, 64 V columns, rows blockIdx.y, + gridDim.y, ....
template <typename T, bool Sums>
__global__ __launch_bounds__(256) void prepare_kernel(PrepareArgs a) {
  using S = typename T::storage;
  using Z = Saved<T>;
  constexpr int V = kVec<T>;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = (static_cast<int>(blockIdx.x) * 64 + lane) * V;
  float sums[V];
#pragma unroll
  for (int i = 0; i < V; ++i) sums[i] = 0.f;
  // Two rows at a time, for their loads to be on their way together.
  const int64_t stride = static_cast<int64_t>(gridDim.y) * 4;
  for (int64_t row = blockIdx.y * 4 + wave; row < a.rows; row += 2 * stride) {
    const bool two = row + stride < a.rows;
    U32x4 raw[2], saved[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (u == 1 && !two) break;
      const int64_t r = row + u * stride;
      raw[u] = load_row<T>(static_cast<const S*>(a.src) + r * a.src_stride, c, a.cols);
      if (a.saved != nullptr)
        saved[u] = load_row<Z>(static_cast<const typename Z::storage*>(a.saved) + r * a.cols, c, a.cols);
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (u == 1 && !two) break;
      float f[V];
      to_floats<T>(raw[u], f);
      U32x4 rounded = raw[u];
      if (a.saved != nullptr) {
        float zf[V];
        to_floats<Z>(saved[u], zf);
        slope_times<T>(zf, a.act, f);
        rounded = from_floats<T>(f);
      }
      if constexpr (Sums) {
#pragma unroll
        for (int i = 0; i < V; ++i) sums[i] += c + i < a.cols ? f[i] : 0.f;
      }
      if (a.out != nullptr && c < a.ld) store16(rounded, static_cast<S*>(a.out) + (row + u * stride) * a.ld + c);
    }
  }
  if constexpr (Sums) {
    __shared__ float area[4][V][64];
#pragma unroll
    for (int i = 0; i < V; ++i) area[wave][i][lane] = sums[i];
    __syncthreads();
    if (wave == 0) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float s = ((area[0][i][lane] + area[1][i][lane]) + area[2][i][lane]) + area[3][i][lane];
        if (c + i < a.cols) a.partial[static_cast<int64_t>(blockIdx.y) * a.cols + c + i] = s;
      }
    }
  }
}

int64_t padded(int64_t cols) { return (cols + 7) / 8 * 8; }

// Rows blocks of a prepare: about four workgroups a compute unit, eight rows each at least.
int prepare_blocks(int dtype, int64_t rows, int64_t cols) {
  const int64_t across = (cols + 64 * (dtype == F32::code ? 4 : 8) - 1) / (64 * (dtype == F32::code ? 4 : 8));
  const int64_t want = (4 * compute_units() + across - 1) / across;
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(want, (rows + 7) / 8)));
}

hipError_t launch_prepare(const PrepareArgs& a, int dtype, int blocks, hipStream_t stream) {
  const int v = dtype == F32::code ? 4 : 8;
  const int64_t width = a.out != nullptr ? std::max<int64_t>(a.ld, a.cols) : a.cols;
  const dim3 grid(static_cast<uint32_t>((width + 64 * v - 1) / (64 * v)), static_cast<uint32_t>(blocks));
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    if (a.partial != nullptr) prepare_kernel<T, true><<<grid, dim3(256), 0, stream>>>(a);
    else prepare_kernel<T, false><<<grid, dim3(256), 0, stream>>>(a);
    return hipGetLastError();
  });
}

// Takes pieces of a workspace; without one it only adds up their sizes.
class Workspace {
 public:
  explicit Workspace(void* base) : base_(static_cast<char*>(base)) {}
  template <typename E>
  E* take(int64_t count) {
    const int64_t at = used_;
    used_ += (count * static_cast<int64_t>(sizeof(E)) + 255) / 256 * 256;
    return base_ != nullptr ? reinterpret_cast<E*>(base_ + at) : nullptr;
  }
  bool dry() const { return base_ == nullptr; }
  int64_t used() const { return used_; }

 private:
  char* base_;
  int64_t used_ = 0;
};

// An operand as the products read it.
struct Laid {
  const void* data;
  int64_t ld;
};

// Whether the products read [rows, cols] as it is.
bool as_it_is(const void* data, int64_t stride, int64_t cols, int dtype) {
  if (dtype == F32::code) return true;
  return reinterpret_cast<uintptr_t>(data) % 16 == 0 && cols % 8 == 0 && stride % 8 == 0 && stride < kMostStride;
}

// `data` as it is, or laid out anew in the workspace.
hipError_t lay_out(const void* data, int64_t stride, int64_t rows, int64_t cols, int dtype, Workspace& ws, Laid& got,
                   hipStream_t stream) {
  if (as_it_is(data, stride, cols, dtype)) {
    got = {data, stride};
    return hipSuccess;
  }
  PrepareArgs p{};
  p.src = data;
  p.src_stride = stride;
  p.ld = padded(cols);
  p.out = ws.take<uint16_t>(rows * p.ld);
  p.rows = rows;
  p.cols = static_cast<int>(cols);
  got = {p.out, p.ld};
  return ws.dry() ? hipSuccess : launch_prepare(p, dtype, prepare_blocks(dtype, rows, cols), stream);
}

template <typename P>
P* rows_on(P* p, int64_t bytes) {
  return p != nullptr ? reinterpret_cast<P*>(reinterpret_cast<uintptr_t>(p) + bytes) : nullptr;
}

// The product `p` of operands a and b, in as many launches as its rows need.
hipError_t multiply(const ProductArgs& p, const Laid& a, const Laid& b, int dtype, bool a_cols, bool b_cols,
                    Workspace& ws, hipStream_t stream) {
  const int64_t size = dtype == F32::code ? 4 : 2;  // of the saved sums as well
  // A in columns is a weight's gradient, with fewer than 2^22 rows.
  return in_slices(p.m, a_cols ? p.m : most_product_rows(p.n), [&](int64_t first, int64_t count) {
    ProductArgs part = p;
    part.m = static_cast<int>(count);
    part.a = rows_on(a.data, first * a.ld * size);
    part.lda = a.ld;
    part.b = b.data;
    part.ldb = b.ld;
    part.residual = rows_on(p.residual, first * p.ldr * size);
    part.saved = rows_on(p.saved, first * p.n * size);
    part.out = rows_on(p.out, first * p.n * size);
    plan_product(part, dtype, a_cols, b_cols);
    if (part.slices > 1) part.partial = ws.take<float>(static_cast<int64_t>(part.slices) * part.m * part.n);
    return ws.dry() ? hipSuccess : launch_product(part, dtype, a_cols, b_cols, stream);
  });
}

}  // namespace

hipError_t launch_linear(const LinearArgs& a, void* workspace, int64_t* bytes, hipStream_t stream) {
  Workspace ws(workspace);
  Laid x, w;
  hipError_t err = lay_out(a.x, a.x_stride, a.rows, a.cols, a.dtype, ws, x, stream);
  if (err == hipSuccess) err = lay_out(a.weight, a.w_stride, a.outs, a.cols, a.dtype, ws, w, stream);
  if (err != hipSuccess) return err;
  ProductArgs p{};
  p.m = static_cast<int>(a.rows);
  p.n = static_cast<int>(a.outs);
  p.k = static_cast<int>(a.cols);
  p.bias = a.bias;
  p.bias_f32 = a.bias_dtype == F32::code;
  p.residual = a.residual;
  p.ldr = a.r_stride;
  p.act = a.act;
  p.saved = a.saved;
  p.out = a.y;
  err = multiply(p, x, w, a.dtype, false, false, ws, stream);
  if (bytes != nullptr) *bytes = ws.used();
  return err;
}

hipError_t launch_linear_backward(const LinearArgs& a, void* workspace, int64_t* bytes, hipStream_t stream) {
  Workspace ws(workspace);
  const bool products = a.dx != nullptr || a.dweight != nullptr;
  // dz, and the column sums for db.
  Laid dz{a.grad, a.g_stride};
  const bool form = products && (a.saved != nullptr || !as_it_is(a.grad, a.g_stride, a.outs, a.dtype));
  if (form || a.dbias != nullptr) {
    const int blocks = prepare_blocks(a.dtype, a.rows, a.outs);
    PrepareArgs p{};
    p.src = a.grad;
    p.src_stride = a.g_stride;
    p.saved = a.saved;
    p.act = a.act;
    p.rows = a.rows;
    p.cols = static_cast<int>(a.outs);
    if (form) {
      p.ld = padded(a.outs);
      p.out = ws.take<char>(a.rows * p.ld * (a.dtype == F32::code ? 4 : 2));
      dz = {p.out, p.ld};
    }
    if (a.dbias != nullptr) p.partial = ws.take<float>(static_cast<int64_t>(blocks) * a.outs);
    if (!ws.dry()) {
      hipError_t err = launch_prepare(p, a.dtype, blocks, stream);
      if (err == hipSuccess && a.dbias != nullptr)
        err = launch_column_sums(p.partial, blocks, a.outs, a.outs, a.dbias, nullptr, a.bias_dtype, stream);
      if (err != hipSuccess) return err;
    }
  }
  hipError_t err = hipSuccess;
  if (a.dx != nullptr) {
    Laid w;
    err = lay_out(a.weight, a.w_stride, a.outs, a.cols, a.dtype, ws, w, stream);
    ProductArgs p{};
    p.m = static_cast<int>(a.rows);
    p.n = static_cast<int>(a.cols);
    p.k = static_cast<int>(a.outs);
    p.out = a.dx;
    if (err == hipSuccess) err = multiply(p, dz, w, a.dtype, false, true, ws, stream);
  }
  if (err == hipSuccess && a.dweight != nullptr) {
    Laid x;
    err = lay_out(a.x, a.x_stride, a.rows, a.cols, a.dtype, ws, x, stream);
    ProductArgs p{};
    p.m = static_cast<int>(a.outs);
    p.n = static_cast<int>(a.cols);
    p.k = static_cast<int>(a.rows);
    p.out = a.dweight;
    if (err == hipSuccess) err = multiply(p, dz, x, a.dtype, true, true, ws, stream);
  }
  if (bytes != nullptr) *bytes = ws.used();
  return err;
}

}  // namespace fh
