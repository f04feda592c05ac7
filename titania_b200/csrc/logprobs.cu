// logprobs.cu — log probabilities of given tokens, the entropy of each row of
// logits and its most likely alternatives (tb200_scorer).
//
// With m the row's largest logit and the others' sum S = Σ' exp(l - m) and
// T = Σ' (m - l) exp(l - m) (Σ' leaves the largest itself out):
//
//     log Z    = log1p(S)                  (relative to m)
//     logprob  = (l - m) - log Z
//     entropy  = log Z + T / (1 + S)
//
// Both terms of the entropy are positive and log1p keeps S's relative error,
// so neither loses digits when one token has almost all of the probability.
#include <algorithm>
#include <string>

#include "runtime.h"

struct tb200_scorer {
  tb200_device* dev = nullptr;
  size_t rows = 0, vocab = 0;
  int top = 0;
  float *logprob = nullptr, *entropy = nullptr, *top_logprobs = nullptr;
  uint32_t* top_ids = nullptr;
  uint32_t* tokens = nullptr;  // [rows] ids given in host memory
};

namespace tb {
namespace {

constexpr int kScoreThreads = 512;
constexpr int kScoreMaxTop = 64;

// The softmax of a set of logits: its largest m, and the sums S and T above
// over the others. An empty set has m = -inf.
struct Soft {
  float m, s, t;
};
// Joins two sets; d <= 0 is the difference of their largest logits.
__device__ __forceinline__ Soft soft_join(const Soft a, const Soft b) {
  const bool a_big = !(b.m > a.m);
  const Soft hi = a_big ? a : b, lo = a_big ? b : a;
  const float d = lo.m - hi.m;
  const float e = expf(d);
  if (!(e > 0.0f) || lo.m == -INFINITY) return hi;  // adds nothing (d may be -inf, or no number)
  Soft r;
  r.m = hi.m;
  r.s = hi.s + e * (1.0f + lo.s);
  r.t = hi.t + e * (lo.t - d * (1.0f + lo.s));
  return r;
}

// One block per row. The alternatives: k passes, each the largest key below the last.
__global__ void __launch_bounds__(kScoreThreads) k_score(const float* __restrict__ logits, int vocab,
                                                         const uint32_t* __restrict__ tokens, int top, float* logprob,
                                                         float* entropy, uint32_t* top_ids, float* top_logprobs) {
  __shared__ Soft red[kScoreThreads / 32];
  __shared__ unsigned long long red_k[kScoreThreads / 32];
  const size_t row = blockIdx.x;
  const float* l = logits + row * vocab;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  Soft a{-INFINITY, 0.f, 0.f};
  bool bad = false;  // a NaN or +inf
  for (int i = threadIdx.x; i < vocab; i += blockDim.x) {
    const float v = l[i];
    bad |= !(v < INFINITY);
    a = soft_join(a, Soft{v, 0.f, 0.f});
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    a = soft_join(a, Soft{__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.s, o),
                          __shfl_xor_sync(0xffffffffu, a.t, o)});
  if (lane == 0) red[warp] = a;
  bad = __syncthreads_or(bad);
  a = red[0];
  for (int w = 1; w < kScoreThreads / 32; w++) a = soft_join(a, red[w]);
  const float nan = __int_as_float(0x7FC00000);
  bad |= a.m == -INFINITY;
  const float logz = bad ? nan : log1pf(a.s);
  if (threadIdx.x == 0) {
    entropy[row] = logz + a.t / (1.0f + a.s);
    const uint32_t tok = tokens[row];
    logprob[row] = tok < uint32_t(vocab) ? (l[tok] - a.m) - logz : nan;
  }
  unsigned long long last = ~0ull;
  for (int k = 0; k < top; k++) {
    unsigned long long best = 0;
    for (int i = threadIdx.x; i < vocab; i += blockDim.x) {
      const unsigned long long key = argmax_key(l[i], uint32_t(i));
      if (key < last && key > best) best = key;
    }
    best = warp_umax64(best);
    __syncthreads();
    if (lane == 0) red_k[warp] = best;
    __syncthreads();
    for (int w = 0; w < kScoreThreads / 32; w++) best = max(best, red_k[w]);
    last = best;
    if (threadIdx.x == 0) {
      const uint32_t id = argmax_index(best);
      top_ids[row * top + k] = id;
      top_logprobs[row * top + k] = (l[id] - a.m) - logz;
    }
  }
}

}  // namespace
}  // namespace tb

extern "C" {

int tb200_scorer_new(tb200_device* dev, size_t rows, size_t vocab, size_t top, tb200_scorer** out) {
  ARG_CHECK(dev && out, "null argument");
  ARG_CHECK(rows >= 1 && rows <= (size_t(1) << 24), "bad number of rows");
  ARG_CHECK(vocab >= 1 && vocab < (size_t(1) << 31), "bad vocabulary");
  ARG_CHECK(top <= size_t(tb::kScoreMaxTop) && top <= vocab, "top must be at most 64 and the vocabulary");
  if (int rc = rt::use(dev)) return rc;
  auto* s = new tb200_scorer;
  s->dev = dev;
  s->rows = rows;
  s->vocab = vocab;
  s->top = int(top);
  cudaError_t e = cudaMalloc(&s->logprob, rows * 4);
  if (e == cudaSuccess) e = cudaMalloc(&s->entropy, rows * 4);
  if (e == cudaSuccess) e = cudaMalloc(&s->tokens, rows * 4);
  if (e == cudaSuccess && top) e = cudaMalloc(&s->top_ids, rows * top * 4);
  if (e == cudaSuccess && top) e = cudaMalloc(&s->top_logprobs, rows * top * 4);
  if (e == cudaSuccess) e = cudaMemsetAsync(s->logprob, 0, rows * 4, dev->stream);
  if (e == cudaSuccess) e = cudaMemsetAsync(s->entropy, 0, rows * 4, dev->stream);
  if (e == cudaSuccess && top) e = cudaMemsetAsync(s->top_ids, 0, rows * top * 4, dev->stream);
  if (e == cudaSuccess && top) e = cudaMemsetAsync(s->top_logprobs, 0, rows * top * 4, dev->stream);
  if (e != cudaSuccess) {
    tb200_scorer_free(s);
    cudaGetLastError();
    return rt::fail(TB200_ERR_CUDA, std::string("scorer: ") + cudaGetErrorString(e));
  }
  *out = s;
  return TB200_OK;
}

int tb200_scorer_free(tb200_scorer* s) {
  if (!s) return TB200_OK;
  cudaSetDevice(s->dev->ordinal);
  cudaStreamSynchronize(s->dev->stream);
  cudaFree(s->logprob);
  cudaFree(s->entropy);
  cudaFree(s->tokens);
  cudaFree(s->top_ids);
  cudaFree(s->top_logprobs);
  delete s;
  return TB200_OK;
}

int tb200_score_enqueue(tb200_scorer* s, const tb200_buffer* logits, const uint32_t* tokens, size_t n) {
  ARG_CHECK(s && logits && (tokens || !n), "null argument");
  ARG_CHECK(n <= s->rows, "score: a scorer of " + std::to_string(s->rows) + " rows can't hold " + std::to_string(n));
  ARG_CHECK(logits->len >= n * s->vocab, "score: the logits buffer holds fewer than rows x vocabulary values");
  if (int rc = rt::use(s->dev)) return rc;
  if (!n) return TB200_OK;
  cudaStream_t st = s->dev->stream;
  cudaPointerAttributes pa{};
  const bool known = cudaPointerGetAttributes(&pa, tokens) == cudaSuccess;
  if (!known) cudaGetLastError();  // a pointer CUDA does not know is host memory
  const bool on_device = known && (pa.type == cudaMemoryTypeDevice || pa.type == cudaMemoryTypeManaged);
  if (on_device) {
    ARG_CHECK(pa.type != cudaMemoryTypeDevice || pa.device == s->dev->ordinal,
              "score: the tokens are in another device's memory");
  } else {
    for (size_t i = 0; i < n; i++)
      ARG_CHECK(tokens[i] < s->vocab, "score: token " + std::to_string(tokens[i]) + " is past the vocabulary of " +
                                          std::to_string(s->vocab));
    cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
    CUDA_TRY(cudaStreamIsCapturing(st, &cap));
    ARG_CHECK(cap == cudaStreamCaptureStatusNone, "score: a captured call needs its tokens in device memory");
    CUDA_TRY(cudaMemcpyAsync(s->tokens, tokens, n * 4, cudaMemcpyHostToDevice, st));
    tokens = s->tokens;
  }
  tb::k_score<<<unsigned(n), tb::kScoreThreads, 0, st>>>(logits->ptr, int(s->vocab), tokens, s->top, s->logprob,
                                                         s->entropy, s->top_ids, s->top_logprobs);
  return rt::launched("score");
}

int tb200_score(tb200_scorer* s, const tb200_buffer* logits, const uint32_t* tokens, size_t n, float* logprob,
                float* entropy, uint32_t* top_ids, float* top_logprobs) {
  if (int rc = tb200_score_enqueue(s, logits, tokens, n)) return rc;
  cudaStream_t st = s->dev->stream;
  const size_t k = n * size_t(s->top);
  if (logprob && n) CUDA_TRY(cudaMemcpyAsync(logprob, s->logprob, n * 4, cudaMemcpyDeviceToHost, st));
  if (entropy && n) CUDA_TRY(cudaMemcpyAsync(entropy, s->entropy, n * 4, cudaMemcpyDeviceToHost, st));
  if (top_ids && k) CUDA_TRY(cudaMemcpyAsync(top_ids, s->top_ids, k * 4, cudaMemcpyDeviceToHost, st));
  if (top_logprobs && k) CUDA_TRY(cudaMemcpyAsync(top_logprobs, s->top_logprobs, k * 4, cudaMemcpyDeviceToHost, st));
  return rt::settle(s->dev);
}

int tb200_scorer_data(const tb200_scorer* s, float** logprob, float** entropy, uint32_t** top_ids,
                      float** top_logprobs) {
  ARG_CHECK(s && logprob && entropy && top_ids && top_logprobs, "null argument");
  *logprob = s->logprob;
  *entropy = s->entropy;
  *top_ids = s->top_ids;
  *top_logprobs = s->top_logprobs;
  return TB200_OK;
}

}  // extern "C"
