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
// by, the scale, and r / scale.
struct RowScale {
  double r, step, c;
  float c32;
  bool zero;  // every integer is 0 (a zero or non-finite row)
  bool fast;  // c32 can be used: nothing near f32's limits
};
__device__ __forceinline__ RowScale row_scale(unsigned long long amax_bits, double r, float* scale_out) {
  RowScale k;
  const double amax = __longlong_as_double(static_cast<long long>(amax_bits));
  float s = float(amax * r / 127.0);
  if (!(s <= 3.402823466e38f)) s = __int_as_float(0x7FC00000);  // NaN for NaN and infinity
  *scale_out = s;
  k.r = r;
  k.zero = !(s > 0.0f);
  k.step = double(s);
  k.c = k.zero ? 0.0 : r / k.step;
  k.c32 = float(k.c);
  k.fast = k.zero || (amax > 0x1p-100 && amax < 0x1p100 && s > 0x1p-100f);
  return k;
}
// The integer of a value v (before the factor r): rint(v r / step), by a product
// with r / step except next to the middle of two integers, where the
// product's last bits would decide.
__device__ __forceinline__ int row_int(double v, const RowScale& k) {
  const double d = v * k.c;
  double q = rint(d);
  if (fabs(fabs(d - q) - 0.5) < 1e-9) q = rint(v * k.r / k.step);
  q = fmin(fmax(q, -127.0), 127.0);
  return k.zero ? 0 : int(q);
}

// Four consecutive values of a row of f32 or bf16, zeros past its end. With
// rows that do not start on vector boundaries, value by value: the same
// sectors, more instructions.
template <bool VEC>
__device__ __forceinline__ float4 load4(const float* p, int left) {
  if (VEC) return *reinterpret_cast<const float4*>(p);
  return make_float4(p[0], left > 1 ? p[1] : 0.f, left > 2 ? p[2] : 0.f, left > 3 ? p[3] : 0.f);
}
template <bool VEC>
__device__ __forceinline__ uint2 load4(const uint16_t* p, int left) {
  if (VEC) return *reinterpret_cast<const uint2*>(p);
  const uint32_t a = p[0], b = left > 1 ? p[1] : 0, c = left > 2 ? p[2] : 0, d = left > 3 ? p[3] : 0;
  return make_uint2(a | (b << 16), c | (d << 16));
}
__device__ __forceinline__ float4 widen(uint2 u) {
  return make_float4(bf_lo(u.x), bf_hi(u.x), bf_lo(u.y), bf_hi(u.y));
}
template <bool VEC>
__device__ __forceinline__ void store4(float* p, int left, float4 v) {
  if (VEC) {
    *reinterpret_cast<float4*>(p) = v;
  } else {
    p[0] = v.x;
    if (left > 1) p[1] = v.y;
    if (left > 2) p[2] = v.z;
    if (left > 3) p[3] = v.w;
  }
}

// A row per `warps` warps (blockDim.x = 32 warps, blockDim.y rows a block),
// E groups of four values a thread, held in registers between the pass that
// finds the scale and the one that rounds.
//
// What bounds it is memory, so the 64-bit work is kept small: only the sum of
// squares takes a conversion per value. The largest |h w| is found among the
// f32 products first (rounding keeps order), then exactly among the few that
// round to it. The integers come from f32 products, whose error is below
// 127 * 2^-22 = 3.1e-5 of a step (three roundings and c32's); only a value
// that near to the middle of two integers is computed again in 64 bits.
template <int SRC, int E, bool VEC>
__global__ void __launch_bounds__(1024) k_rows_q8(RowArgs a, long long rows) {
  constexpr bool kNorm = SRC == kRowNorm || SRC == kRowAddNorm;
  __shared__ double red_s[32];
  __shared__ unsigned long long red_m[32];
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, warps = blockDim.x >> 5;
  const long long row = (long long)blockIdx.x * blockDim.y + threadIdx.y;
  if (row >= rows) return;  // only where a row is one warp: no barrier below
  const float* xf = static_cast<const float*>(a.x) + row * a.cols;
  const uint16_t* xh = static_cast<const uint16_t*>(a.x) + row * a.cols;

  float4 h[E];
  uint2 w[E];  // bf16
#pragma unroll
  for (int i = 0; i < E; i++) {
    const int at = 4 * (tid + i * blockDim.x), left = a.cols - at;
    h[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    w[i] = make_uint2(0, 0);
    if (left <= 0) continue;
    if constexpr (SRC == kRowBf16)
      h[i] = widen(load4<VEC>(xh + at, left));
    else
      h[i] = load4<VEC>(xf + at, left);
    if constexpr (kNorm) w[i] = load4<VEC>(a.w + at, left);
  }
  if constexpr (SRC == kRowAddNorm) {
#pragma unroll
    for (int i = 0; i < E; i++) {
      const int at = 4 * (tid + i * blockDim.x), left = a.cols - at;
      if (left <= 0) continue;
      const float4 y = load4<VEC>(a.y + row * a.cols + at, left);
      h[i] = make_float4(__fadd_rn(h[i].x, y.x), __fadd_rn(h[i].y, y.y), __fadd_rn(h[i].z, y.z),
                         __fadd_rn(h[i].w, y.w));
      store4<VEC>(const_cast<float*>(xf) + at, left, h[i]);
    }
  }

  double ss = 0.0;
  float m32 = 0.f;
#pragma unroll
  for (int i = 0; i < E; i++) {
    const float4 wf = widen(w[i]);
    const float v[4] = {h[i].x, h[i].y, h[i].z, h[i].w}, u[4] = {wf.x, wf.y, wf.z, wf.w};
#pragma unroll
    for (int j = 0; j < 4; j++) {
      if (kNorm) {
        const double d = double(v[j]);
        ss = fma(d, d, ss);
      }
      const float p = fabsf(kNorm ? __fmul_rn(v[j], u[j]) : v[j]);
      m32 = p <= m32 ? m32 : p;  // a NaN stays
    }
  }
  unsigned long long amax = 0;
#pragma unroll
  for (int i = 0; i < E; i++) {
    const float4 wf = widen(w[i]);
    const float v[4] = {h[i].x, h[i].y, h[i].z, h[i].w}, u[4] = {wf.x, wf.y, wf.z, wf.w};
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const float p = fabsf(kNorm ? __fmul_rn(v[j], u[j]) : v[j]);
      if (!(p < m32)) amax = max(amax, abs_bits(kNorm ? double(v[j]) * double(u[j]) : double(v[j])));
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    if (kNorm) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  }
  if (warps > 1) {  // one row a block
    if ((tid & 31) == 0) {
      red_s[tid >> 5] = ss;
      red_m[tid >> 5] = amax;
    }
    __syncthreads();
    const int l = tid & 31;
    ss = l < warps ? red_s[l] : 0.0;
    amax = l < warps ? red_m[l] : 0ull;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      if (kNorm) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    }
  }
  const double r = kNorm ? 1.0 / sqrt(ss / double(a.cols) + a.eps) : 1.0;
  float s;
  const RowScale k = row_scale(amax, r, &s);
  if (tid == 0) a.scale[row] = s;
  int8_t* q = a.q + row * a.ld;
#pragma unroll
  for (int i = 0; i < E; i++) {
    const int at = 4 * (tid + i * blockDim.x);
    if (at >= a.ld) continue;  // the padding gets its zeros: values past the row's end are 0
    const float4 wf = widen(w[i]);
    const float v[4] = {h[i].x, h[i].y, h[i].z, h[i].w}, u[4] = {wf.x, wf.y, wf.z, wf.w};
    uint32_t b[4];
    bool sure = k.fast;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const float d = __fmul_rn(kNorm ? __fmul_rn(v[j], u[j]) : v[j], k.c32);
      const float t = __fadd_rn(d, 12582912.0f);  // 1.5 * 2^23: the sum's low bits are the rounded integer
      b[j] = __float_as_uint(t);
      sure = sure && fabsf(__fsub_rn(d, __fsub_rn(t, 12582912.0f))) < 0.4999f;
    }
    if (!sure && !k.zero) {
#pragma unroll
      for (int j = 0; j < 4; j++) b[j] = uint32_t(row_int(kNorm ? double(v[j]) * double(u[j]) : double(v[j]), k));
    }
    uint32_t word = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    if (k.zero) word = 0;
    *reinterpret_cast<uint32_t*>(q + at) = word;
  }
}

// Rows too long for registers: one block per row, read twice (h from x, where
// the first pass left it).
template <int SRC>
__global__ void __launch_bounds__(1024) k_long_rows_q8(RowArgs a) {
  constexpr bool kNorm = SRC == kRowNorm || SRC == kRowAddNorm;
  __shared__ double red_s[32];
  __shared__ unsigned long long red_m[32];
  pdl_launch_dependents();
  pdl_wait();
  const size_t row = blockIdx.x;
  float* xf = static_cast<float*>(const_cast<void*>(a.x)) + row * a.cols;
  const uint16_t* xh = static_cast<const uint16_t*>(a.x) + row * a.cols;
  double ss = 0.0;
  unsigned long long amax = 0;
  for (int i = threadIdx.x; i < a.cols; i += blockDim.x) {
    double v;
    if constexpr (SRC == kRowBf16) {
      v = double(bf16f(xh[i]));
    } else {
      float h = xf[i];
      if (SRC == kRowAddNorm) xf[i] = h = __fadd_rn(h, a.y[row * a.cols + i]);
      v = double(h);
      if (kNorm) {
        ss = fma(v, v, ss);
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
  for (int i = 0; i < 32; i++) {
    ss += red_s[i];
    amax = max(amax, red_m[i]);
  }
  const double r = kNorm ? 1.0 / sqrt(ss / double(a.cols) + a.eps) : 1.0;
  float s;
  const RowScale k = row_scale(amax, r, &s);
  if (threadIdx.x == 0) a.scale[row] = s;
  int8_t* q = a.q + row * a.ld;
  for (int i = threadIdx.x; i < a.ld; i += blockDim.x) {
    double v = 0.0;
    if (i < a.cols) {
      v = SRC == kRowBf16 ? double(bf16f(xh[i])) : double(xf[i]);
      if (kNorm) v *= double(bf16f(a.w[i]));
    }
    q[i] = int8_t(row_int(v, k));
  }
}

// Four values a thread; blockDim.x threads along a row, blockDim.y rows.
template <bool VEC>
__global__ void __launch_bounds__(256) k_dequantize(float* __restrict__ out, const int8_t* __restrict__ q,
                                                    const float* __restrict__ scale, long long rows, int cols, int ld) {
  pdl_launch_dependents();
  pdl_wait();
  const long long row = (long long)blockIdx.x * blockDim.y + threadIdx.y;
  if (row >= rows) return;
  const float s = scale[row];
  for (int at = 4 * (threadIdx.x + blockIdx.y * blockDim.x); at < cols; at += 4 * blockDim.x * gridDim.y) {
    const char4 v = *reinterpret_cast<const char4*>(q + row * ld + at);
    store4<VEC>(out + row * cols + at, cols - at,
                make_float4(__fmul_rn(float(v.x), s), __fmul_rn(float(v.y), s), __fmul_rn(float(v.z), s),
                            __fmul_rn(float(v.w), s)));
  }
}

template <int SRC>
void launch_rows_q8(tb200_device* d, const RowArgs& a, size_t rows) {
  // Threads that have four values each; the padding (fewer than 16) is theirs too.
  const int groups = a.ld / 4;
  const bool vec = a.cols % 4 == 0;
  // Few rows: as many threads on each as it has groups, since what counts is
  // how long one row takes. Many: several groups a thread, so that more of a
  // row's loads are in flight at once and its reduction is shared by fewer warps.
  const bool few = rows < size_t(2 * d->sms);
  int e = 1;
  while (e < 4 && groups > e * (few ? 1024 : 128)) e *= 2;
  if (groups > e * 1024) {
    launch_pdl(k_long_rows_q8<SRC>, dim3(unsigned(rows)), dim3(1024), 0, d->stream, a);
    return;
  }
  const int tx = (groups + 32 * e - 1) / (32 * e) * 32, ty = tx == 32 ? 4 : 1;
  const dim3 grid(unsigned((rows + ty - 1) / ty)), block(tx, ty);
#define TB_ROWS(E)                                                                               \
  if (e == E) {                                                                                  \
    if (vec)                                                                                     \
      launch_pdl(k_rows_q8<SRC, E, true>, grid, block, 0, d->stream, a, (long long)rows);        \
    else                                                                                         \
      launch_pdl(k_rows_q8<SRC, E, false>, grid, block, 0, d->stream, a, (long long)rows);       \
  }
  TB_ROWS(1)
  TB_ROWS(2)
  TB_ROWS(4)
#undef TB_ROWS
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
  tb::launch_rows_q8<tb::kRowF32>(d, a, out->rows);
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
    tb::launch_rows_q8<tb::kRowBf16>(d, a, q->rows);
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
  const size_t groups = (x->cols + 3) / 4;
  unsigned tx = 32;
  while (tx < 256 && tx < groups) tx *= 2;
  const unsigned ty = 256 / tx;
  const dim3 grid(unsigned((x->rows + ty - 1) / ty), unsigned(std::min<size_t>((groups + tx - 1) / tx, 65535)));
  if (x->cols % 4 == 0)
    tb::launch_pdl(tb::k_dequantize<true>, grid, dim3(tx, ty), 0, d->stream, out->ptr, x->values, x->scales,
                   (long long)x->rows, int(x->cols), int(x->ld));
  else
    tb::launch_pdl(tb::k_dequantize<false>, grid, dim3(tx, ty), 0, d->stream, out->ptr, x->values, x->scales,
                   (long long)x->rows, int(x->cols), int(x->ld));
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
    tb::launch_rows_q8<tb::kRowAddNorm>(d, a, out->rows);
  else
    tb::launch_rows_q8<tb::kRowNorm>(d, a, out->rows);
  return rt::launched("add_rmsnorm_q8");
}

}  // extern "C"
