// q8.cu — rows of 8-bit integers with an f32 scale each (tb200_q8): the
// handle, and the kernels that turn f32 or bf16 rows into such rows and back.
//
// A row n_0 .. n_{C-1} becomes s = f32(max|n| / 127), q_i = rint(n_i / s). Three
// sources give the n_i:
//   tb200_quantize         n = x (f32)
//   tb200_quantize_weight  n = w (bf16), a row per output channel
//   tb200_add_rmsnorm_q8   h = f32(x + y), stored back to x;
//                          n = h * w / sqrt(mean(h^2) + eps)
// All of it after the f32 addition is 64-bit arithmetic. h * w (24 + 8 bits) and
// h^2 (48 bits) are exact there, so which integer a value next to the middle of
// two becomes does not depend on the order of a sum, on the number of threads
// or on how a compiler contracts a product: the rows are the same, bit for
// bit, whatever variant runs, and equal those of any 64-bit restatement.
#include <algorithm>
#include <string>

#include "runtime.h"

namespace tb {
namespace {

enum RowSource { kRowF32, kRowBf16, kRowNorm, kRowAddNorm };

struct RowArgs {
  const void* x;      // [rows][cols] f32 (bf16: kRowBf16); kRowAddNorm: also written
  const float* y;     // kRowAddNorm: [rows][cols]
  const uint16_t* w;  // norm weight [cols]
  double eps;
  int8_t* q;          // [rows][ld]
  float* scale;       // [rows]
  int cols, ld;
};

// |v| as an integer that orders as |v| does, with every NaN above infinity.
__device__ __forceinline__ unsigned long long abs_bits(double v) {
  return static_cast<unsigned long long>(__double_as_longlong(v)) & 0x7FFFFFFFFFFFFFFFull;
}

// What a row's values have in common: the factor r that each is multiplied
// by, the scale and r / scale.
struct RowScale {
  double r, step, c;
  bool zero;  // every integer is 0 (a zero or non-finite row)
};
__device__ __forceinline__ RowScale row_scale(double ss, unsigned long long amax, double r, float* scale_out) {
  RowScale k;
  k.r = r;
  float s = float(__longlong_as_double(static_cast<long long>(amax)) * r / 127.0);
  if (!(s <= 3.402823466e38f)) s = __int_as_float(0x7FC00000);  // NaN for NaN and infinity
  *scale_out = s;
  k.zero = !(s > 0.0f);
  k.step = double(s);
  k.c = k.zero ? 0.0 : r / k.step;
  return k;
}
// The integer of a value v (before the factor r): rint(v r / step), by a product
// with r / step except next to the middle of two integers, where the
// product's last bits would decide.
__device__ __forceinline__ int row_int(double v, const RowScale& k) {
  double d = v * k.c;
  double q = rint(d);
  if (fabs(fabs(d - q) - 0.5) < 1e-9) q = rint(v * k.r / k.step);
  q = fmin(fmax(q, -127.0), 127.0);
  return k.zero ? 0 : int(q);
}

// One block per row; the row is read twice.
template <int SRC>
__global__ void __launch_bounds__(256) k_rows_q8(RowArgs a) {
  __shared__ double red_s[8];
  __shared__ unsigned long long red_m[8];
  const size_t row = blockIdx.x;
  const float* xf = static_cast<const float*>(a.x) + row * a.cols;
  const uint16_t* xh = static_cast<const uint16_t*>(a.x) + row * a.cols;
  double ss = 0.0;
  unsigned long long amax = 0;
  for (int i = threadIdx.x; i < a.cols; i += blockDim.x) {
    double v;
    if (SRC == kRowBf16) {
      v = double(bf16f(xh[i]));
    } else {
      float h = xf[i];
      if (SRC == kRowAddNorm) {
        h = __fadd_rn(h, a.y[row * a.cols + i]);
        const_cast<float*>(xf)[i] = h;
      }
      v = double(h);
      if (SRC >= kRowNorm) {
        ss += v * v;
        v *= double(bf16f(a.w[i]));
      }
    }
    amax = max(amax, abs_bits(v));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    ss += __shfl_xor_sync(0xffffffffu, ss, o);
    amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  }
  if ((threadIdx.x & 31) == 0) {
    red_s[threadIdx.x >> 5] = ss;
    red_m[threadIdx.x >> 5] = amax;
  }
  __syncthreads();
  ss = 0.0;
  amax = 0;
  for (int i = 0; i < 8; i++) {
    ss += red_s[i];
    amax = max(amax, red_m[i]);
  }
  const double r = SRC >= kRowNorm ? 1.0 / sqrt(ss / double(a.cols) + a.eps) : 1.0;
  float s;
  const RowScale k = row_scale(ss, amax, r, &s);
  if (threadIdx.x == 0) a.scale[row] = s;
  int8_t* q = a.q + row * a.ld;
  for (int i = threadIdx.x; i < a.ld; i += blockDim.x) {
    if (i >= a.cols) {
      q[i] = 0;
      continue;
    }
    double v = SRC == kRowBf16 ? double(bf16f(xh[i])) : double(xf[i]);
    if (SRC >= kRowNorm) v *= double(bf16f(a.w[i]));
    q[i] = int8_t(row_int(v, k));
  }
}

__global__ void k_dequantize(float* __restrict__ out, const int8_t* __restrict__ q, const float* __restrict__ scale,
                             int cols, int ld) {
  const size_t row = blockIdx.x;
  const float s = scale[row];
  for (int i = threadIdx.x; i < cols; i += blockDim.x) out[row * cols + i] = __fmul_rn(float(q[row * ld + i]), s);
}

template <int SRC>
void launch_rows_q8(cudaStream_t s, const RowArgs& a, size_t rows) {
  k_rows_q8<SRC><<<unsigned(rows), 256, 0, s>>>(a);
}

RowArgs row_args(const tb200_q8* out) {
  RowArgs a{};
  a.q = out->values;
  a.scale = out->scales;
  a.cols = int(out->cols);
  a.ld = int(out->ld);
  return a;
}

}  // namespace
}  // namespace tb

namespace {

constexpr size_t kMaxDim = (size_t(1) << 31) - 1;

void q8_release(tb200_q8* q) {
  cudaFree(q->values);
  cudaFree(q->scales);
  delete q;
}

}  // namespace

extern "C" {

int tb200_q8_new(tb200_device* d, size_t rows, size_t cols, tb200_q8** out) {
  if (int rc = rt::use(d)) return rc;
  ARG_CHECK(out, "null output handle");
  ARG_CHECK(cols > 0 && cols <= kMaxDim - 15, "q8: bad number of columns");
  ARG_CHECK(rows <= kMaxDim, "q8: too many rows");
  auto* q = new tb200_q8;
  q->rows = q->cap = rows;
  q->cols = cols;
  q->ld = (cols + 15) / 16 * 16;
  if (rows) {
    cudaError_t e = cudaMalloc(&q->values, rows * q->ld);
    if (e == cudaSuccess) e = cudaMalloc(&q->scales, rows * 4);
    if (e == cudaSuccess) e = cudaMemsetAsync(q->values, 0, rows * q->ld, d->stream);
    if (e == cudaSuccess) e = cudaMemsetAsync(q->scales, 0, rows * 4, d->stream);
    if (e != cudaSuccess) {
      q8_release(q);
      cudaGetLastError();  // reported here; not left for the next launch check
      return rt::fail(TB200_ERR_CUDA, std::string("q8: ") + cudaGetErrorString(e));
    }
  }
  *out = q;
  return TB200_OK;
}

int tb200_q8_free(tb200_device* d, tb200_q8* q) {
  if (!q) return TB200_OK;
  if (int rc = rt::use(d)) return rc;
  CUDA_TRY(cudaStreamSynchronize(d->stream));
  q8_release(q);
  return TB200_OK;
}

int tb200_q8_resize(tb200_device* d, tb200_q8* q, size_t rows) {
  if (int rc = rt::use(d)) return rc;
  ARG_CHECK(q, "null argument");
  ARG_CHECK(rows <= q->cap, "8-bit rows made for " + std::to_string(q->cap) + " can't hold " + std::to_string(rows));
  q->rows = rows;
  return TB200_OK;
}

int tb200_q8_shape(const tb200_q8* q, size_t* rows, size_t* cols) {
  ARG_CHECK(q && rows && cols, "null argument");
  *rows = q->rows;
  *cols = q->cols;
  return TB200_OK;
}

int tb200_q8_read(tb200_device* d, const tb200_q8* q, int8_t* values, float* scales) {
  if (int rc = rt::use(d)) return rc;
  ARG_CHECK(q && ((values && scales) || !q->rows), "null argument");
  if (q->rows) {
    CUDA_TRY(cudaMemcpy2DAsync(values, q->cols, q->values, q->ld, q->cols, q->rows, cudaMemcpyDeviceToHost, d->stream));
    CUDA_TRY(cudaMemcpyAsync(scales, q->scales, q->rows * 4, cudaMemcpyDeviceToHost, d->stream));
  }
  return rt::settle(d);
}

int tb200_q8_write(tb200_device* d, tb200_q8* q, const int8_t* values, const float* scales) {
  if (int rc = rt::use(d)) return rc;
  ARG_CHECK(q && ((values && scales) || !q->rows), "null argument");
  if (q->rows) {
    CUDA_TRY(cudaMemcpy2DAsync(q->values, q->ld, values, q->cols, q->cols, q->rows, cudaMemcpyHostToDevice, d->stream));
    CUDA_TRY(cudaMemcpyAsync(q->scales, scales, q->rows * 4, cudaMemcpyHostToDevice, d->stream));
  }
  return rt::settle(d);
}

int tb200_q8_data(const tb200_q8* q, int8_t** values, size_t* ld, float** scales) {
  ARG_CHECK(q && values && ld && scales, "null argument");
  *values = q->values;
  *ld = q->ld;
  *scales = q->scales;
  return TB200_OK;
}

int tb200_quantize(tb200_device* d, tb200_q8* out, const tb200_buffer* x) {
  if (int rc = rt::use(d)) return rc;
  ARG_CHECK(out && x, "null argument");
  ARG_CHECK(x->len == out->rows * out->cols, "quantize: input holds " + std::to_string(x->len) + " values, expected " +
                                                 std::to_string(out->rows * out->cols));
  if (!out->rows) return TB200_OK;
  tb::RowArgs a = tb::row_args(out);
  a.x = x->ptr;
  tb::launch_rows_q8<tb::kRowF32>(d->stream, a, out->rows);
  return rt::launched("quantize");
}

int tb200_quantize_weight(tb200_device* d, const tb200_weight* w, tb200_q8** out) {
  if (int rc = rt::use(d)) return rc;
  ARG_CHECK(w && out, "null argument");
  ARG_CHECK(w->shape.size() == 2, "quantize_weight: weight is not a matrix");
  tb200_q8* q = nullptr;
  if (int rc = tb200_q8_new(d, w->shape[0], w->shape[1], &q)) return rc;
  if (q->rows) {
    tb::RowArgs a = tb::row_args(q);
    a.x = w->ptr;
    tb::launch_rows_q8<tb::kRowBf16>(d->stream, a, q->rows);
    if (int rc = rt::launched("quantize_weight")) {
      q8_release(q);
      return rc;
    }
  }
  *out = q;
  return TB200_OK;
}

int tb200_dequantize(tb200_device* d, tb200_buffer* out, const tb200_q8* x) {
  if (int rc = rt::use(d)) return rc;
  ARG_CHECK(out && x, "null argument");
  ARG_CHECK(out->len == x->rows * x->cols, "dequantize: output holds " + std::to_string(out->len) +
                                               " values, expected " + std::to_string(x->rows * x->cols));
  if (!x->rows) return TB200_OK;
  tb::k_dequantize<<<unsigned(x->rows), 256, 0, d->stream>>>(out->ptr, x->values, x->scales, int(x->cols), int(x->ld));
  return rt::launched("dequantize");
}

int tb200_add_rmsnorm_q8(tb200_device* d, tb200_q8* out, tb200_buffer* x, const tb200_buffer* y,
                         const tb200_weight* w, float eps) {
  if (int rc = rt::use(d)) return rc;
  ARG_CHECK(out && x && w, "null argument");
  ARG_CHECK(x != y, "add_rmsnorm_q8: x and y are the same buffer");
  const size_t n = out->rows * out->cols;
  ARG_CHECK(x->len == n, "add_rmsnorm_q8: x holds " + std::to_string(x->len) + " values, expected " + std::to_string(n));
  ARG_CHECK(!y || y->len == n,
            "add_rmsnorm_q8: y holds " + std::to_string(y ? y->len : 0) + " values, expected " + std::to_string(n));
  ARG_CHECK(w->numel == out->cols, "add_rmsnorm_q8: weight holds " + std::to_string(w->numel) + " values, expected " +
                                       std::to_string(out->cols));
  ARG_CHECK(eps >= 0.0f, "add_rmsnorm_q8: eps must not be negative");
  if (!out->rows) return TB200_OK;
  tb::RowArgs a = tb::row_args(out);
  a.x = x->ptr;
  a.y = y ? y->ptr : nullptr;
  a.w = w->ptr;
  a.eps = double(eps);
  if (y)
    tb::launch_rows_q8<tb::kRowAddNorm>(d->stream, a, out->rows);
  else
    tb::launch_rows_q8<tb::kRowNorm>(d->stream, a, out->rows);
  return rt::launched("add_rmsnorm_q8");
}

}  // extern "C"
