// q8.cu — rows of 8-bit integers with an f32 scale each (tb200_q8): the
// handle, and the kernels that turn f32 or bf16 rows into such rows and back.
//
// A row n_0 .. n_{C-1} becomes s = f32(max|n| / 127), q_i = rint(n_i / s). Three
// sources give the n_i:
//   tb200_quantize         n = x (f32)
//   tb200_quantize_weight  n = w (bf16), a row per output channel
//   tb200_add_rmsnorm_q8   h = f32(x + y), stored back to x;
//                          n = h * w / sqrt(mean(h^2) + eps)
// All of it after the f32 addition is 64-bit arithmetic, in which h * w (24 + 8
// bits) and h^2 (48 bits) are exact. Rows of f32 and bf16 are therefore the same,
// bit for bit, whatever variant runs, and equal those of any 64-bit restatement. A
// norm's sum of squares is rounded in an order that the variant sets (the numbers of
// rows and columns choose it), and its mean and square root round once each: the row's
// factor agrees with another order's to a few times 1e-15 (up to 16384 columns; the
// bound grows with them), so only a value that near to the middle of two integers, or a scale
// that near to the middle of two f32 values, may come out as the other one.
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
  double eps, inv_cols;
  int8_t* q;          // [rows][ld]
  float* scale;       // [rows]
  int cols, ld;
};

// |v| as an integer that orders as |v| does, with every NaN above infinity.
__device__ __forceinline__ unsigned long long abs_bits(double v) {
  return static_cast<unsigned long long>(__double_as_longlong(v)) & 0x7FFFFFFFFFFFFFFFull;
}

// What a row's values have in common: the factor r that each is multiplied by
// and the scale.
struct RowScale {
  double r, c;      // c: r / s to a few units of 2^-48
  float s;
  float c32, sure;  // f32 products with c32 this near to an integer round as they have to
};
__device__ __forceinline__ RowScale row_scale(double amax, double r) {
  RowScale k;
  k.r = r;
  // The product with 1 / 127 is within 2^-52 of the quotient. Of an f32 amax (r = 1) the quotient
  // is never that near to the middle of two f32 values, so its rounding is the quotient's.
  k.s = float(amax * r * (1.0 / 127.0));
  if (!(k.s <= 3.402823466e38f)) k.s = __int_as_float(0x7FC00000);  // NaN for NaN and infinity
  const bool plain = amax > 0x1p-100 && amax < 0x1p100 && k.s > 0x1p-100f && k.s < 0x1p100f;
  // One Newton step from the f32 reciprocal, which a division in 64 bits would take three of.
  const double s = plain ? double(k.s) : 1.0, i = double(__frcp_rn(float(s)));
  k.c = r * fma(i, fma(-s, i, 1.0), i);
  k.c32 = float(k.c);
  k.sure = plain ? 0.49995f : -1.0f;  // near f32's limits every integer is computed by a quotient
  return k;
}
// rint(v r / s), the integer of a value v (before the factor r), in 64 bits.
__device__ __noinline__ int row_int(double v, double r, float s) {
  if (!(s > 0.0f)) return 0;  // zeros, or no numbers
  return int(fmin(fmax(rint(v * r / double(s)), -127.0), 127.0));
}
// The same by a product, except next to the middle of two integers.
__device__ __forceinline__ int row_int(double v, const RowScale& k) {
  if (!(k.s > 0.0f)) return 0;
  const double d = v * k.c, q = rint(d);
  return k.sure > 0.f && fabs(fabs(d - q) - 0.5) > 1e-9 ? int(q) : row_int(v, k.r, k.s);
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

// The largest of |a| and b, a NaN if there is one.
__device__ __forceinline__ float max_abs(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(fabsf(a)), "f"(b));
  return r;
}
// The largest of the lanes' 64-bit numbers.
__device__ __forceinline__ unsigned long long warp_max64(unsigned long long v) {
  const unsigned hi = __reduce_max_sync(0xffffffffu, unsigned(v >> 32));
  const unsigned lo = __reduce_max_sync(0xffffffffu, unsigned(v >> 32) == hi ? unsigned(v) : 0u);
  return (static_cast<unsigned long long>(hi) << 32) | lo;
}

// The most threads of a block, by its threads' groups: what leaves them the registers.
__host__ __device__ constexpr int row_threads(int e) { return e == 8 ? 512 : e == 4 ? 640 : 1024; }

// A row per blockDim.x / 32 warps (blockDim.y rows a block), E groups of four
// values a thread, held in registers between the pass that finds the scale and
// the one that rounds.
//
// Every warp of a row repeats what a row costs beside its values (the two
// reductions, the constants): 5003 x 2560 with the residual takes 46, 33 and
// 30 us with one, two and four groups a thread (31.4 over several buffers in turns, 5.3 TB/s).
//
// What should bound it is memory, so the 64-bit work is kept small (with all of
// it in 64 bits the kernel took 51 instructions a value): only the sum of
// squares takes a conversion per value. The largest |h w| is found among the
// f32 products first (rounding keeps order), then exactly by the threads that
// hold it. The integers come from f32 products, whose error is below 127 * 2^-22
// = 3.1e-5 of a step (h w, the product and c32 round once each); only a value
// that near to the middle of two integers is computed again in 64 bits.
template <int SRC, int E, bool VEC>
__global__ void __launch_bounds__(row_threads(E)) k_rows_q8(RowArgs a, long long rows) {
  constexpr bool kNorm = SRC == kRowNorm || SRC == kRowAddNorm;
  __shared__ double red_s[32];
  __shared__ unsigned red_m[32];
  __shared__ unsigned long long exact;
  pdl_launch_dependents();
  const int tid = threadIdx.x, warps = blockDim.x >> 5, lane = tid & 31;
  const long long row = (long long)blockIdx.x * blockDim.y + threadIdx.y;
  if (tid == 0 && warps > 1) exact = 0;
  pdl_wait();
  if (row >= rows) return;  // only where a row is one warp: no barrier below
  const float* xf = static_cast<const float*>(a.x) + row * a.cols;
  const uint16_t* xh = static_cast<const uint16_t*>(a.x) + row * a.cols;

  float4 h[E], y[E];
  uint2 w[E];  // bf16
#pragma unroll
  for (int i = 0; i < E; i++) {
    const int at = 4 * (tid + i * blockDim.x), left = a.cols - at;
    h[i] = y[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    w[i] = make_uint2(0, 0);
    if (left <= 0) continue;
    if constexpr (SRC == kRowBf16)
      h[i] = widen(load4<VEC>(xh + at, left));
    else
      h[i] = load4<VEC>(xf + at, left);
    if constexpr (SRC == kRowAddNorm) y[i] = load4<VEC>(a.y + row * a.cols + at, left);
    if constexpr (kNorm) w[i] = load4<VEC>(a.w + at, left);
  }
  // What is rounded, before the row's factor: h w in f32, or the value itself.
  auto products = [&](int i, float (&p)[4]) {
    const float4 u = kNorm ? widen(w[i]) : make_float4(1.f, 1.f, 1.f, 1.f);
    p[0] = kNorm ? __fmul_rn(h[i].x, u.x) : h[i].x;
    p[1] = kNorm ? __fmul_rn(h[i].y, u.y) : h[i].y;
    p[2] = kNorm ? __fmul_rn(h[i].z, u.z) : h[i].z;
    p[3] = kNorm ? __fmul_rn(h[i].w, u.w) : h[i].w;
  };
  // The same exactly.
  auto value = [&](int i, int j) {
    const float4 u = kNorm ? widen(w[i]) : make_float4(1.f, 1.f, 1.f, 1.f);
    const float v[4] = {h[i].x, h[i].y, h[i].z, h[i].w}, f[4] = {u.x, u.y, u.z, u.w};
    return kNorm ? double(v[j]) * double(f[j]) : double(v[j]);
  };
  double ss = 0.0;
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < E; i++) {
    const int at = 4 * (tid + i * blockDim.x), left = a.cols - at;
    if constexpr (SRC == kRowAddNorm) {
      h[i] = make_float4(__fadd_rn(h[i].x, y[i].x), __fadd_rn(h[i].y, y[i].y), __fadd_rn(h[i].z, y[i].z),
                         __fadd_rn(h[i].w, y[i].w));
      if (left > 0) store4<VEC>(const_cast<float*>(xf) + at, left, h[i]);
    }
    if constexpr (kNorm) {
      const double d0 = h[i].x, d1 = h[i].y, d2 = h[i].z, d3 = h[i].w;
      ss = fma(d0, d0, ss), ss = fma(d1, d1, ss), ss = fma(d2, d2, ss), ss = fma(d3, d3, ss);
    }
    float p[4];
    products(i, p);
    m = max_abs(p[3], max_abs(p[2], max_abs(p[1], max_abs(p[0], m))));
  }
  unsigned top = __reduce_max_sync(0xffffffffu, __float_as_uint(m));  // as integers: NaN above infinity
  if (kNorm) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  }
  if (warps > 1) {  // one row a block
    if (lane == 0) {
      red_s[tid >> 5] = ss;
      red_m[tid >> 5] = top;
    }
    __syncthreads();
    top = __reduce_max_sync(0xffffffffu, lane < warps ? red_m[lane] : 0u);
    if (kNorm) {
      // Each group of `span` lanes (a power of two, at least the number of warps) adds the warps' sums.
      const int span = 1 << (32 - __clz(warps - 1));
      ss = (lane & (span - 1)) < warps ? red_s[lane & (span - 1)] : 0.0;
      for (int o = span / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    }
  }
  double amax = double(__uint_as_float(top));
  if (kNorm) {
    // Exactly, of the products that round to the largest.
    unsigned long long best = 0;
    if (__float_as_uint(m) == top) {
#pragma unroll
      for (int i = 0; i < E; i++) {
        float p[4];
        products(i, p);
#pragma unroll
        for (int j = 0; j < 4; j++)
          if (fabsf(p[j]) == m) best = max(best, abs_bits(value(i, j)));
      }
    }
    if (warps > 1) {
      if (best) atomicMax(&exact, best);
      __syncthreads();
      best = exact;
    } else {
      best = warp_max64(best);
    }
    if (!isnan(__uint_as_float(top))) amax = __longlong_as_double(static_cast<long long>(best));
  }
  const RowScale k = row_scale(amax, kNorm ? rsqrt(fma(ss, a.inv_cols, a.eps)) : 1.0);
  if (tid == 0) a.scale[row] = k.s;
  int8_t* q = a.q + row * a.ld;
#pragma unroll
  for (int i = 0; i < E; i++) {
    const int at = 4 * (tid + i * blockDim.x);
    if (at >= a.ld) continue;  // the padding gets its zeros: values past the row's end are 0
    float p[4];
    products(i, p);
    uint32_t b[4];
    float off = 0.f;  // the largest distance from an integer
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const float d = __fmul_rn(p[j], k.c32);
      const float t = __fadd_rn(d, 12582912.0f);  // 1.5 * 2^23: the sum's low bits are the rounded integer
      b[j] = __float_as_uint(t);
      off = max_abs(__fsub_rn(d, __fsub_rn(t, 12582912.0f)), off);
    }
    if (!(off < k.sure)) {
#pragma unroll
      for (int j = 0; j < 4; j++) b[j] = uint32_t(row_int(value(i, j), k));
    }
    *reinterpret_cast<uint32_t*>(q + at) =
        __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
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
  const double r = kNorm ? rsqrt(fma(ss, a.inv_cols, a.eps)) : 1.0;
  const RowScale k = row_scale(__longlong_as_double(static_cast<long long>(amax)), r);
  if (threadIdx.x == 0) a.scale[row] = k.s;
  int8_t* q = a.q + row * a.ld;
  for (int i = threadIdx.x; i < a.ld; i += blockDim.x) {
    double v = 0.0;
    if (i < a.cols) {
      v = SRC == kRowBf16 ? double(bf16f(xh[i])) : double(xf[i]);
      if (kNorm) v *= double(bf16f(a.w[i]));
    }
    q[i] = int8_t(row_int(v, r, k.s));
  }
}

// Groups of four values (the aligned ones of the output, whose
// rows begin `shift` values after one where `cols` is no multiple of four: an
// unaligned store4 each took 5000 x 2562 from 10.7 to 22 us in L2; from memory 16.2), kDeq of them
// a thread, so that a thread has more than one word on its way; blockDim.x
// threads along a row, blockDim.y rows.
constexpr int kDeq = 4;
__global__ void __launch_bounds__(256) k_dequantize(float* out, const int8_t* q, const float* scale, long long rows,
                                                    int cols, int ld) {
  pdl_launch_dependents();
  pdl_wait();
  const long long row = (long long)blockIdx.x * blockDim.y + threadIdx.y;
  if (row >= rows) return;
  const int shift = int((row * cols) & 3), groups = (cols + shift + 3) / 4;
  const uint32_t* words = reinterpret_cast<const uint32_t*>(q + row * ld);
  float* to = out + row * cols;
  for (int g0 = threadIdx.x + kDeq * blockDim.x * blockIdx.y; g0 < groups; g0 += kDeq * blockDim.x * gridDim.y) {
    uint32_t v[kDeq];
#pragma unroll
    for (int i = 0; i < kDeq; i++) {
      const int g = g0 + i * blockDim.x;
      if (g >= groups) continue;
      v[i] = 4 * g < ld ? words[g] : 0;
      if (shift) v[i] = __funnelshift_l(g ? words[g - 1] : 0, v[i], 8 * shift);
    }
    const float s = scale[row];
#pragma unroll
    for (int i = 0; i < kDeq; i++) {
      const int g = g0 + i * blockDim.x, at = 4 * g - shift;
      if (g >= groups) continue;
      const float4 x = make_float4(float(int8_t(v[i])), float(int8_t(v[i] >> 8)), float(int8_t(v[i] >> 16)),
                                   float(int8_t(v[i] >> 24)));
      const float4 y = make_float4(__fmul_rn(x.x, s), __fmul_rn(x.y, s), __fmul_rn(x.z, s), __fmul_rn(x.w, s));
      if (at >= 0 && at + 4 <= cols) {
        *reinterpret_cast<float4*>(to + at) = y;
      } else {
        const float e[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int j = 0; j < 4; j++)
          if (at + j >= 0 && at + j < cols) to[at + j] = e[j];
      }
    }
  }
}

template <int SRC>
void launch_rows_q8(tb200_device* d, const RowArgs& a, size_t rows) {
  constexpr bool kNorm = SRC == kRowNorm || SRC == kRowAddNorm;
  const int groups = a.ld / 4;  // of four values; the padding is theirs too
  // Few rows: as many threads on each as it has groups, since what counts is how
  // long one row takes. Many: as few warps as can hold it, one if it fits, up to
  // four groups a thread with a norm, eight without (2048 x 9728, one buffer: 31 and 17 us with
  // four and eight, 18.9 from memory; with the residual and the norm 54 and 83, for want of registers).
  int e = 1;
  if (rows >= size_t(2 * d->sms))
    while (e < (kNorm ? 4 : 8) && groups > e * 32) e *= 2;
  while (e < 8 && groups > e * row_threads(e)) e *= 2;
  if (groups > e * row_threads(e)) {
    launch_pdl(k_long_rows_q8<SRC>, dim3(unsigned(rows)), dim3(1024), 0, d->stream, a);
    return;
  }
  const int tx = (groups + 32 * e - 1) / (32 * e) * 32, ty = tx == 32 ? 4 : 1;
  const dim3 grid(unsigned((rows + ty - 1) / ty)), block(tx, ty);
  const bool vec = a.cols % 4 == 0;
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
  TB_ROWS(8)
#undef TB_ROWS
}

RowArgs row_args(const tb200_q8* out) {
  RowArgs a{};
  a.q = out->values;
  a.scale = out->scales;
  a.cols = int(out->cols);
  a.inv_cols = 1.0 / double(out->cols);
  a.ld = int(out->ld);
  return a;
}

}  // namespace
}  // namespace tb

namespace {

constexpr size_t kMaxDim = size_t(1) << 30;  // 32-bit indices along a row, and of rows in tiles

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
  ARG_CHECK(cols > 0 && cols <= kMaxDim, "q8: bad number of columns");
  ARG_CHECK(rows <= kMaxDim, "q8: too many rows");
  auto* q = new tb200_q8;
  q->dev = d;
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
  ARG_CHECK(rt::of(d, q), "free: the 8-bit rows were made on another device");
  CUDA_TRY(cudaStreamSynchronize(d->stream));
  q8_release(q);
  return TB200_OK;
}

int tb200_q8_resize(tb200_device* d, tb200_q8* q, size_t rows) {
  if (int rc = rt::use(d)) return rc;
  ARG_CHECK(q, "null argument");
  ARG_CHECK(rt::of(d, q), "resize: the 8-bit rows were made on another device");
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
  ARG_CHECK(rt::of(d, q), "the 8-bit rows were made on another device");
  if (q->rows) {
    CUDA_TRY(cudaMemcpy2DAsync(values, q->cols, q->values, q->ld, q->cols, q->rows, cudaMemcpyDeviceToHost, d->stream));
    CUDA_TRY(cudaMemcpyAsync(scales, q->scales, q->rows * 4, cudaMemcpyDeviceToHost, d->stream));
  }
  return rt::settle(d);
}

int tb200_q8_write(tb200_device* d, tb200_q8* q, const int8_t* values, const float* scales) {
  if (int rc = rt::use(d)) return rc;
  ARG_CHECK(q && ((values && scales) || !q->rows), "null argument");
  ARG_CHECK(rt::of(d, q), "the 8-bit rows were made on another device");
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
  ARG_CHECK(rt::of(d, out, x), "quantize: an operand was made on another device");
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
  ARG_CHECK(rt::of(d, w), "quantize_weight: the weight was made on another device");
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
  ARG_CHECK(rt::of(d, out, x), "dequantize: an operand was made on another device");
  ARG_CHECK(out->len == x->rows * x->cols, "dequantize: output holds " + std::to_string(out->len) +
                                               " values, expected " + std::to_string(x->rows * x->cols));
  if (!x->rows) return TB200_OK;
  const size_t groups = (x->cols + (x->cols % 4 ? 3 : 0) + 3) / 4;
  // Few rows: a group a thread, as many threads as there are; many: kDeq groups a thread.
  const size_t each = x->rows * groups < size_t(d->sms) * 2048 ? 1 : tb::kDeq;
  unsigned tx = 32;
  while (tx < 256 && tx * each < groups) tx *= 2;
  const unsigned ty = 256 / tx;
  const size_t along = (groups + tx * tb::kDeq - 1) / (tx * tb::kDeq);
  const dim3 grid(unsigned((x->rows + ty - 1) / ty), unsigned(std::min<size_t>(along, 65535)));
  tb::launch_pdl(tb::k_dequantize, grid, dim3(tx, ty), 0, d->stream, out->ptr, x->values, x->scales,
                 (long long)x->rows, int(x->cols), int(x->ld));
  return rt::launched("dequantize");
}

int tb200_add_rmsnorm_q8(tb200_device* d, tb200_q8* out, tb200_buffer* x, const tb200_buffer* y,
                         const tb200_weight* w, float eps) {
  if (int rc = rt::use(d)) return rc;
  ARG_CHECK(out && x && w, "null argument");
  ARG_CHECK(rt::of(d, out, x, y, w), "add_rmsnorm_q8: an operand was made on another device");
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
