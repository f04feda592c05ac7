// logprobs.cu — log probabilities of given tokens, the entropy of each row of
// logits and its most likely alternatives (tb200_scorer).
//
// With m the row's largest logit and the others' sums S = Σ' exp(l - m) and
// T = Σ' (m - l) exp(l - m) (Σ' leaves the largest itself out):
//
//     log Z    = log1p(S)                  (relative to m)
//     logprob  = (l - m) - log Z
//     entropy  = log Z + T / (1 + S)
//
// Both terms of the entropy are positive and log1p keeps S's relative error,
// so neither loses digits when one token has almost all of the probability.
//
// One launch, one pass over the logits, bound by reading them. A row is cut
// into chunks, a CTA each (few rows) or several rows' chunks fill the GPU
// (many). A warp takes 128 logits (a block) at a time: their largest, one
// redux, is both the running maximum that the sums refer to, so that rescaling
// is a rare warp-uniform branch, and the block's entry in a table of 1/128 of
// the logits' size. The last CTA of a row joins the chunks' sums and finds
// the alternatives: the k largest logits lie in the k blocks with the largest
// maxima (each of those has an element at least as large as any element of
// another block), so only those blocks are read again.
#include <algorithm>
#include <string>

#include "runtime.h"

struct tb200_scorer {
  tb200_device* dev = nullptr;
  size_t rows = 0, vocab = 0;
  int top = 0;
  float *logprob = nullptr, *entropy = nullptr, *top_logprobs = nullptr;
  uint32_t* top_ids = nullptr;
  uint32_t* tokens = nullptr;   // [rows] ids given in host memory
  float4* part = nullptr;       // sums of the chunks
  int* block_max = nullptr;     // [rows][blocks], when there are alternatives
  unsigned* ticket = nullptr;   // [rows], zero between launches
};

namespace tb {
namespace {

constexpr int kScoreThreads = 256;
constexpr int kScoreWarps = kScoreThreads / 32;
constexpr int kScoreMaxTop = 64;
constexpr int kBlock = 128;        // logits per warp step and table entry
constexpr int kUnroll = 4;         // blocks a warp has in flight
constexpr int kCand = 1024;        // candidates ranked in shared memory
constexpr int kOwn = 8;            // table entries a thread keeps in registers
constexpr int kNegInf = int(0xFF800000u ^ 0x7FFFFFFFu);  // order(-inf)
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// IEEE total order as a signed integer (argmax_key's order), and back.
__device__ __forceinline__ int order(float v) {
  const int b = __float_as_int(v);
  return b ^ int(uint32_t(b >> 31) >> 1);
}
__device__ __forceinline__ float unorder(int o) { return __int_as_float(o ^ int(uint32_t(o >> 31) >> 1)); }
// An ordered value and an index as one key: larger is preferred, ties to the lower index.
__device__ __forceinline__ unsigned long long order_key(int o, uint32_t i) {
  return (static_cast<unsigned long long>(uint32_t(o) ^ 0x80000000u) << 32) | (0xFFFFFFFFu - i);
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The softmax of a set of logits: its largest m, and the sums above over the
// others; t in units of log 2. An empty set has m = -inf.
struct Soft {
  float m, s, t;
};
// `a` seen from a larger maximum m: its own largest joins the others.
__device__ __forceinline__ Soft soft_under(const Soft a, float m) {
  const float d = (m - a.m) * kLog2e, e = ex2(-d);
  if (e == 0.0f) return Soft{m, 0.0f, 0.0f};  // d may be infinite
  const float s = fmaf(e, a.s, e);
  return Soft{m, s, fmaf(e, a.t, d * s)};
}
__device__ __forceinline__ Soft soft_join(const Soft a, const Soft b) {
  const bool a_big = !(b.m > a.m);
  const Soft hi = a_big ? a : b, lo = a_big ? b : a;
  if (lo.m == -INFINITY) return Soft{hi.m, hi.s + lo.s, hi.t};  // nothing, or the NaN that it met
  const Soft u = soft_under(lo, hi.m);
  return Soft{hi.m, hi.s + u.s, hi.t + u.t};
}

// The row as blocks of 128 logits that start on 16-byte boundaries: element
// 4 g + j - shift of the row is value j of granule g, and lane i of a warp has
// granule 32 b + i of block b. The first and last granule may reach over the row's ends.
struct Row {
  const float* base;  // of granule 0
  int shift, vocab, blocks;
  __device__ __forceinline__ Row(const float* logits, size_t row, int vocab_) : vocab(vocab_) {
    const size_t at = row * size_t(vocab);
    shift = int(at & 3);
    base = logits + (at - shift);
    blocks = (vocab + shift + kBlock - 1) / kBlock;
  }
  __device__ __forceinline__ bool inside(int b) const { return b * kBlock >= shift && (b + 1) * kBlock <= vocab + shift; }
  // Element i of the row for value j of lane's granule of block b, or out of range.
  __device__ __forceinline__ int element(int b, int lane, int j) const { return b * kBlock + 4 * lane + j - shift; }
  __device__ __forceinline__ float4 load(int b, int lane) const {
    return __ldg(reinterpret_cast<const float4*>(base) + size_t(b) * 32 + lane);
  }
  // A block at the row's end: `fill` in the place of what is not the row's.
  __device__ __forceinline__ float4 load_end(int b, int lane, float fill) const {
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int i = element(b, lane, j);
      v[j] = i >= 0 && i < vocab ? __ldg(base + size_t(b) * kBlock + 4 * lane + j) : fill;
    }
    return make_float4(v[0], v[1], v[2], v[3]);
  }
};

// Adds a block to the warp's set (a.m is the warp's, a.s and a.t each lane's
// share). bm: the block's largest in order.
__device__ __forceinline__ void add_block(Soft& a, float4 v, int bm, int lane) {
  float x[4] = {v.x, v.y, v.z, v.w};
  if (bm <= kNegInf) {  // nothing but excluded tokens; a NaN below them counts
    if (isnan(x[0]) || isnan(x[1]) || isnan(x[2]) || isnan(x[3])) a.s = __int_as_float(0x7FC00000);
    return;
  }
  float skip[4] = {0.f, 0.f, 0.f, 0.f};
  if (bm > order(a.m)) {  // warp-uniform: a new maximum
    const float m = unorder(bm);
    // Lane 0 carries the old maximum's own term; every lane its share of the others'.
    const float d = (m - a.m) * kLog2e, e = ex2(-d);
    if (a.m == -INFINITY) {
      // nothing yet (or a NaN, which stays)
    } else if (e == 0.0f) {
      a.s *= 0.0f;
      a.t = 0.0f;
    } else {
      const float s = lane == 0 ? fmaf(e, a.s, e) : e * a.s;
      a.t = fmaf(e, a.t, d * s);
      a.s = s;
    }
    a.m = m;
    // The maximum itself stays out of the sums: its first place in the block.
    const int mine = order(x[0]) == bm ? 0 : order(x[1]) == bm ? 1 : order(x[2]) == bm ? 2 : order(x[3]) == bm ? 3 : 4;
    const unsigned who = __ballot_sync(0xffffffffu, mine < 4);
    if (lane == __ffs(who) - 1) {
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (j == mine) skip[j] = -INFINITY;
    }
  }
  float e[4], d[4];
#pragma unroll
  for (int j = 0; j < 4; j++) {
    d[j] = (x[j] - a.m) * kLog2e + skip[j];
    e[j] = ex2(d[j]);
    d[j] = fmaxf(d[j], -200.0f);  // 0 * -inf has to be 0
  }
  a.s += (e[0] + e[1]) + (e[2] + e[3]);
  a.t -= fmaf(d[0], e[0], d[1] * e[1]) + fmaf(d[2], e[2], d[3] * e[3]);
}

__device__ __forceinline__ int max4(float4 v) { return max(max(order(v.x), order(v.y)), max(order(v.z), order(v.w))); }

// A key with k <= #{keys >= it} <= most: bisection over 64-bit keys that no
// two entries share. count(key) is called by all threads and is the same for
// all; at least k keys exist.
template <class Count>
__device__ __forceinline__ unsigned long long key_bound(int k, int most, Count count) {
  unsigned long long lo = 0, hi = ~0ull;  // count(lo) >= k; count(hi + 1) < k
  while (lo < hi) {
    const unsigned long long mid = lo + (hi - lo) / 2 + 1;
    const int c = count(mid);
    if (c >= k) {
      lo = mid;
      if (c <= most) break;
    } else {
      hi = mid - 1;
    }
  }
  return lo;
}

struct ScoreArgs {
  const float* logits;
  const uint32_t* tokens;
  float *logprob, *entropy, *top_logprobs;
  uint32_t* top_ids;
  float4* part;     // [rows][chunks]
  int* block_max;   // [rows][max_blocks]
  unsigned* ticket;
  int vocab, top, chunks, chunk_blocks, max_blocks;
};

struct ScoreShared {
  Soft soft[kScoreWarps];
  int last, n_blocks, n_cand;
  int counts[2][kScoreWarps];
  unsigned long long cand[kCand];
  int blocks[kScoreMaxTop + kScoreMaxTop / 2 + 4];
};

// The sum of c over the CTA, on every thread. Calls take `turn` 0, 1, 0, ... in
// turns: a second one cannot overwrite what a slow warp still reads of the first.
__device__ __forceinline__ int cta_sum(int c, int& turn, ScoreShared& sh) {
  c = __reduce_add_sync(0xffffffffu, c);
  int* counts = sh.counts[turn];
  turn ^= 1;
  if ((threadIdx.x & 31) == 0) counts[threadIdx.x >> 5] = c;
  __syncthreads();
  int total = 0;
#pragma unroll
  for (int w = 0; w < kScoreWarps; w++) total += counts[w];
  return total;
}

// The `top` largest of the row, ranked: by the whole CTA.
__device__ void alternatives(const ScoreArgs& a, const Row& r, size_t row, const int* block_max, float m, float logz,
                             ScoreShared& sh) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int k = a.top;
  int turn = 0;
  if (threadIdx.x == 0) sh.n_blocks = sh.n_cand = 0;
  // The blocks with the largest maxima: k of them, or more where that ends the search sooner.
  unsigned long long own[kOwn];
#pragma unroll
  for (int i = 0; i < kOwn; i++) {
    const int b = int(threadIdx.x) + i * kScoreThreads;
    own[i] = b < r.blocks ? order_key(__ldcg(block_max + b), uint32_t(b)) : 0ull;
  }
  const int kb = min(k, r.blocks);
  const unsigned long long bound = key_bound(kb, kb + kb / 2 + 4, [&](unsigned long long key) {
    int c = 0;
#pragma unroll
    for (int i = 0; i < kOwn; i++) c += own[i] >= key;
    for (int b = int(threadIdx.x) + kOwn * kScoreThreads; b < r.blocks; b += kScoreThreads)
      c += order_key(__ldcg(block_max + b), uint32_t(b)) >= key;
    return cta_sum(c, turn, sh);
  });
  __syncthreads();
  auto pick = [&](unsigned long long key, int b) {
    if (key >= bound && key) sh.blocks[atomicAdd(&sh.n_blocks, 1)] = b;
  };
#pragma unroll
  for (int i = 0; i < kOwn; i++) pick(own[i], int(threadIdx.x) + i * kScoreThreads);
  for (int b = int(threadIdx.x) + kOwn * kScoreThreads; b < r.blocks; b += kScoreThreads)
    pick(order_key(__ldcg(block_max + b), uint32_t(b)), b);
  __syncthreads();
  const int nb = sh.n_blocks;
  // f(key) of every element of those blocks.
  auto each = [&](auto f) {
    for (int i = warp; i < nb; i += kScoreWarps) {
      const int b = sh.blocks[i];
      const float4 v = r.inside(b) ? r.load(b, lane) : r.load_end(b, lane, 0.f);
      const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int at = r.element(b, lane, j);
        f(at >= 0 && at < a.vocab ? order_key(order(x[j]), uint32_t(at)) : 0ull);
      }
    }
  };
  // Candidates: the elements at least as large as the smallest of the picked
  // maxima (k of these exist), or all elements where there are fewer blocks than k.
  unsigned long long least = r.blocks < k ? 0ull : bound & 0xFFFFFFFF00000000ull;
  for (int tries = 0; tries < 2; tries++) {
    each([&](unsigned long long key) {
      if (key >= least && key) {
        const int at = atomicAdd(&sh.n_cand, 1);
        if (at < kCand) sh.cand[at] = key;
      }
    });
    __syncthreads();
    if (sh.n_cand <= kCand) break;
    // More than there is room for (neighbours that are all large): a bound that leaves fewer.
    least = key_bound(k, kCand, [&](unsigned long long key) {
      int c = 0;
      each([&](unsigned long long x) { c += x >= key; });
      return cta_sum(c, turn, sh);
    });
    __syncthreads();
    if (threadIdx.x == 0) sh.n_cand = 0;
    __syncthreads();
  }
  const int n = sh.n_cand;
  for (int i = threadIdx.x; i < n; i += kScoreThreads) {
    const unsigned long long mine = sh.cand[i];
    int rank = 0;
    for (int j = 0; j < n; j++) rank += sh.cand[j] > mine;
    if (rank < k) {
      a.top_ids[row * k + rank] = argmax_index(mine);
      a.top_logprobs[row * k + rank] = (unorder(int(uint32_t(mine >> 32) ^ 0x80000000u)) - m) - logz;
    }
  }
}

__global__ void __launch_bounds__(kScoreThreads) k_score(ScoreArgs a) {
  __shared__ ScoreShared sh;
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const size_t row = blockIdx.x / unsigned(a.chunks);
  const int chunk = int(blockIdx.x % unsigned(a.chunks));
  const Row r(a.logits, row, a.vocab);
  int* block_max = a.top ? a.block_max + row * size_t(a.max_blocks) : nullptr;
  const int b0 = chunk * a.chunk_blocks, b1 = min(r.blocks, b0 + a.chunk_blocks);
  Soft s{-INFINITY, 0.f, 0.f};
  for (int b = b0 + warp * kUnroll; b < b1; b += kScoreWarps * kUnroll) {
    float4 v[kUnroll];
    bool in[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; u++) {
      in[u] = b + u < b1 && r.inside(b + u);
      if (in[u]) v[u] = r.load(b + u, lane);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; u++) {
      if (b + u >= b1) break;
      int bm;
      if (in[u]) {
        bm = max4(v[u]);
      } else {
        v[u] = r.load_end(b + u, lane, __int_as_float(-1));  // the lowest in order
        bm = max4(v[u]);
        v[u] = r.load_end(b + u, lane, -INFINITY);
      }
      bm = __reduce_max_sync(0xffffffffu, bm);
      if (block_max && lane == 0) block_max[b + u] = bm;
      add_block(s, v[u], bm, lane);
    }
  }
  s.s = warp_sum(s.s);
  s.t = warp_sum(s.t);
  if (lane == 0) sh.soft[warp] = s;
  __syncthreads();
  s = sh.soft[0];
#pragma unroll
  for (int w = 1; w < kScoreWarps; w++) s = soft_join(s, sh.soft[w]);
  if (a.chunks > 1) {
    if (threadIdx.x == 0) {
      a.part[blockIdx.x] = make_float4(s.m, s.s, s.t, 0.f);
      __threadfence();
      sh.last = atomicAdd(a.ticket + row, 1u) == unsigned(a.chunks) - 1;
      __threadfence();
    }
    __syncthreads();
    if (!sh.last) return;
    // The last CTA of the row: every chunk's sums, in an order that is the same each time.
    Soft p{-INFINITY, 0.f, 0.f};
    for (int c = threadIdx.x; c < a.chunks; c += kScoreThreads) {
      const float4 q = __ldcg(a.part + row * a.chunks + c);
      p = soft_join(p, Soft{q.x, q.y, q.z});
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const Soft q{__shfl_xor_sync(0xffffffffu, p.m, o), __shfl_xor_sync(0xffffffffu, p.s, o),
                   __shfl_xor_sync(0xffffffffu, p.t, o)};
      // The lower lane's set first on both sides, so that both get the same bits.
      p = (lane & o) ? soft_join(q, p) : soft_join(p, q);
    }
    if (lane == 0) sh.soft[warp] = p;
    __syncthreads();
    s = sh.soft[0];
#pragma unroll
    for (int w = 1; w < kScoreWarps; w++) s = soft_join(s, sh.soft[w]);
    if (threadIdx.x == 0) a.ticket[row] = 0;
  }
  const float nan = __int_as_float(0x7FC00000);
  const bool bad = !(s.m < INFINITY) || s.m == -INFINITY || isnan(s.s);
  const float logz = bad ? nan : log1pf(s.s);
  if (threadIdx.x == 0) {
    a.entropy[row] = logz + kLn2 * s.t / (1.0f + s.s);
    const uint32_t tok = a.tokens[row];
    a.logprob[row] = tok < uint32_t(a.vocab) ? (__ldg(r.base + r.shift + tok) - s.m) - logz : nan;
  }
  if (a.top) alternatives(a, r, row, block_max, s.m, logz, sh);
}

// Blocks of a row, whatever its alignment.
int score_blocks(size_t vocab) { return int((vocab + 3 + kBlock - 1) / kBlock); }
// CTAs that a call of n rows aims for: eight resident ones on each SM.
int score_target(const tb200_device* d) { return 8 * d->sms; }
// Chunks per row: one when the rows alone fill the GPU; else enough to, each
// of at least one block for every warp.
int score_chunks(const tb200_device* d, size_t n, int blocks) {
  const size_t want = (size_t(score_target(d)) + n - 1) / n;
  return int(std::max<size_t>(1, std::min<size_t>(want, size_t(blocks + kScoreWarps - 1) / kScoreWarps)));
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
  const int blocks = tb::score_blocks(vocab);
  // n rows in score_chunks(n) chunks: at most n + the CTAs aimed for, and no row has more than blocks.
  const size_t parts = rows + size_t(tb::score_target(dev));
  if (e == cudaSuccess) e = cudaMalloc(&s->part, parts * sizeof(float4));
  if (e == cudaSuccess) e = cudaMalloc(&s->ticket, rows * 4);
  if (e == cudaSuccess) e = cudaMemsetAsync(s->ticket, 0, rows * 4, dev->stream);
  if (e == cudaSuccess && top) e = cudaMalloc(&s->block_max, rows * blocks * 4);
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
  cudaFree(s->part);
  cudaFree(s->block_max);
  cudaFree(s->ticket);
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
  tb::ScoreArgs a{};
  a.logits = logits->ptr;
  a.tokens = tokens;
  a.logprob = s->logprob;
  a.entropy = s->entropy;
  a.top_ids = s->top_ids;
  a.top_logprobs = s->top_logprobs;
  a.part = s->part;
  a.block_max = s->block_max;
  a.ticket = s->ticket;
  a.vocab = int(s->vocab);
  a.top = s->top;
  a.max_blocks = tb::score_blocks(s->vocab);
  a.chunks = tb::score_chunks(s->dev, n, a.max_blocks);
  a.chunk_blocks = (a.max_blocks + a.chunks - 1) / a.chunks;
  a.chunks = (a.max_blocks + a.chunk_blocks - 1) / a.chunk_blocks;
  tb::launch_pdl(tb::k_score, dim3(unsigned(n * a.chunks)), dim3(tb::kScoreThreads), 0, st, a);
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
