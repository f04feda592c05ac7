// q8_gemm.cu — the product of 8-bit rows (tb200_matmul_q8):
//
//     out[t][c] = f32(Σ_k w[c][k] · x[t][k]) · (sw[c] · sx[t])
//
// The sum is exact in 32-bit integers (|q| <= 128 and at most 131071 columns),
// so its order is free; the two f32 roundings of the scales' product and the
// final product follow it.
#include <algorithm>
#include <string>

#include "runtime.h"

namespace tb {
namespace {

constexpr size_t kMaxCols = 131071;  // 128 * 128 * 131071 < 2^31

// One warp per channel and up to 4 tokens.
__global__ void __launch_bounds__(256) k_matvec_q8(float* __restrict__ out, const int8_t* __restrict__ w,
                                                   const float* __restrict__ sw, int channels,
                                                   const int8_t* __restrict__ x, const float* __restrict__ sx,
                                                   int tokens, int ldw, int ldx) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int c = blockIdx.x * 8 + warp, t0 = blockIdx.y * 4;
  if (c >= channels) return;
  int acc[4] = {0, 0, 0, 0};
  const int4* wr = reinterpret_cast<const int4*>(w + size_t(c) * ldw);
  for (int i = lane; i < ldw / 16; i += 32) {
    const int4 a = wr[i];
#pragma unroll
    for (int t = 0; t < 4; t++) {
      if (t0 + t >= tokens) break;
      const int4 b = reinterpret_cast<const int4*>(x + size_t(t0 + t) * ldx)[i];
      acc[t] = __dp4a(a.x, b.x, acc[t]);
      acc[t] = __dp4a(a.y, b.y, acc[t]);
      acc[t] = __dp4a(a.z, b.z, acc[t]);
      acc[t] = __dp4a(a.w, b.w, acc[t]);
    }
  }
#pragma unroll
  for (int t = 0; t < 4; t++) {
    const int s = __reduce_add_sync(0xffffffffu, acc[t]);
    if (lane == t && t0 + t < tokens)
      out[size_t(t0 + t) * channels + c] = __fmul_rn(__int2float_rn(s), __fmul_rn(sw[c], sx[t0 + t]));
  }
}

}  // namespace
}  // namespace tb

extern "C" {

int tb200_matmul_q8(tb200_device* d, tb200_buffer* out, const tb200_q8* w, const tb200_q8* x) {
  if (int rc = rt::use(d)) return rc;
  ARG_CHECK(out && w && x, "null argument");
  ARG_CHECK(w->cols == x->cols, "matmul_q8: weight has " + std::to_string(w->cols) + " columns, input " +
                                    std::to_string(x->cols));
  ARG_CHECK(w->cols <= tb::kMaxCols, "matmul_q8: more than 131071 columns do not sum in 32 bits");
  ARG_CHECK(out->len == x->rows * w->rows, "matmul_q8: output holds " + std::to_string(out->len) + ", expected " +
                                               std::to_string(x->rows * w->rows));
  if (!x->rows || !w->rows) return TB200_OK;
  const dim3 grid(unsigned((w->rows + 7) / 8), unsigned((x->rows + 3) / 4));
  tb::k_matvec_q8<<<grid, 256, 0, d->stream>>>(out->ptr, w->values, w->scales, int(w->rows), x->values, x->scales,
                                               int(x->rows), int(w->ld), int(x->ld));
  return rt::launched("matmul_q8");
}

}  // extern "C"
