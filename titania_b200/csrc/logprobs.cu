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
// One pass over the logits, in steps of 512 of a row, which a warp takes at a time as four blocks of 128. The
// blocks' largest, a redux each, are both the running maximum that the sums refer
// to and their entries in a table of 1/128 of the logits' size. Per logit there
// are five instructions for the sums and one for the maximum; at ten the kernel
// was bound by them (1111 x 151936: 142 us; 108, of which the bytes take 105). Who takes what:
//   k_score_rows       rows of up to four steps: a warp a row, in its registers;
//   k_score_long_rows  many rows of up to 64 steps: a warp a row, step by step;
//   k_score            else: a CTA a row, or a part of one (deal() below). The CTA
//                      that finishes a row's last piece joins the pieces' sums, in
//                      their order.
// The warps of a CTA begin a piece with the largest of their first steps as
// common maximum, so that few steps raise it: that is a warp-uniform branch as
// dear as a step.
//
// The alternatives: the k largest logits lie in the k blocks with the largest
// maxima (each of those has an element at least as large as any element of
// another block), so only those are read again. In k_score that is a few
// microseconds a row, of waiting more than of work: with few rows the CTA that
// finishes a row does it (64 rows, five alternatives: 15.8 us, 11.5 with none, in L2; 17.4 and 13.5 from memory),
// with many it is a kernel of its own with a CTA for every row (1111 rows: 124 us;
// in one kernel 131). One alternative is the maximum itself, whose place the warps
// keep (112 us).
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <climits>
#include <string>

#include "runtime.h"

struct tb200_scorer {
  tb200_device* dev = nullptr;
  size_t rows = 0, vocab = 0;
  int top = 0;
  float *logprob = nullptr, *entropy = nullptr, *top_logprobs = nullptr;
  uint32_t* top_ids = nullptr;
  uint32_t* tokens = nullptr;   // [rows] ids given in host memory
  float4* part = nullptr;       // sums of the pieces
  unsigned long long* part_best = nullptr;  // their largest logits, when there is one alternative
  int* block_max = nullptr;     // [rows][a row's blocks], when there are several
  float2* peak = nullptr;       // [rows] maximum and log Z, likewise
  unsigned* ticket = nullptr;   // [rows], zero between launches
  int ctas = 0;                 // that the GPU runs at once
};

namespace tb {
namespace {

constexpr int kScoreThreads = 256;
constexpr int kScoreWarps = kScoreThreads / 32;
constexpr int kScoreMaxTop = 64;
constexpr int kBlock = 128;        // logits per table entry
constexpr int kStep = 4;           // blocks a warp takes at a time
// Alternatives: a search for the k largest may end with up to this many.
__host__ __device__ constexpr int slack(int k) { return k + k / 2 + 4; }
constexpr int kPicked = slack(kScoreMaxTop);  // blocks read again
constexpr int kCand = 4 * kPicked;            // elements of as many granules
constexpr int kOwn = 8;                       // table entries a thread keeps in registers
constexpr int kGranules = 13;                 // granules of the picked blocks that it keeps
static_assert(kPicked * 32 <= kGranules * kScoreThreads, "they fit");
constexpr int kOneByOne = 6;                  // alternatives of a short row that are found in turn
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

// The softmax of a set of logits under a maximum m that none of them exceeds:
// the sums above, t in units of log 2. own: 1 where m is one of the set's logits,
// which then stands outside the sums, else 0. An empty set may have m = -inf.
struct Soft {
  float m, s, t, own;
};
__device__ __forceinline__ Soft soft_join(const Soft a, const Soft b) {
  const bool a_big = !(b.m > a.m);
  const Soft hi = a_big ? a : b, lo = a_big ? b : a;
  if (lo.m == -INFINITY) return Soft{hi.m, hi.s + lo.s, hi.t, hi.own};  // nothing, or the NaN that it met
  const float d = (hi.m - lo.m) * kLog2e, e = ex2(-d);
  if (d == 0.0f) {  // of two places of the maximum one stays outside
    const float own = fmaxf(hi.own, lo.own);
    return Soft{hi.m, hi.s + lo.s + (hi.own + lo.own - own), hi.t + lo.t, own};
  }
  if (e == 0.0f) return Soft{hi.m, hi.s + lo.s * 0.0f, hi.t, hi.own};  // d may be infinite; a NaN stays
  const float s = e * (lo.s + lo.own);
  return Soft{hi.m, hi.s + s, hi.t + fmaf(e, lo.t, d * s), hi.own};
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
    return ld_f32x4(base + size_t(b) * kBlock + 4 * lane);
  }
  // A block at the row's end: `fill` in the place of what is not the row's.
  __device__ __forceinline__ float4 load_end(int b, int lane, float fill) const {
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int i = element(b, lane, j);
      v[j] = i >= 0 && i < vocab ? ld_f32(base + size_t(b) * kBlock + 4 * lane + j) : fill;
    }
    return make_float4(v[0], v[1], v[2], v[3]);
  }
};

// A warp's set while it grows: m and own are the warp's, s and t each lane's
// shares of the sums, taken at c = f32(m log2 e) in the place of m log2 e, which
// saves an instruction a logit: what that leaves out (lo) is put right in settled().
// A share holds 2^lo and settled() takes it out again, so lo has to be small: up
// to |m| = 2^20 it is at most 2^-4, half a step of c there. Beyond (logits of a finite
// mask value such as -1e10 or -1e30, where a step of c is hundreds and more) the
// shares are taken at m itself, by a subtraction and a product.
struct Running {
  float m, c, lo, s, t;
  int order;  // of m
  bool own;
  __device__ __forceinline__ explicit Running(int o) : s(0.f), t(0.f), own(false) { refer(o); }
  __device__ __forceinline__ void refer(int o) {
    order = o;
    m = unorder(o);
    c = m * kLog2e;
    lo = m > -INFINITY && !far() ? fmaf(m, kLog2e, -c) : 0.f;
  }
  __device__ __forceinline__ bool far() const { return fabsf(m) > 0x1p20f; }
  __device__ __forceinline__ Soft settled() const {
    const float f = ex2(-lo);
    return Soft{m, s * f, fmaf(lo, s, t) * f, own ? 1.f : 0.f};
  }
  // Refers the sums to a larger maximum; lane 0 takes the old one's own term. The
  // old sums are brought to c, where the shares to come are taken: brought to m
  // they were off by 2^lo, which is 1 + 5e-3 at m = 3e5.
  __device__ __forceinline__ void raise(int o, int lane) {
    const Soft old = settled();
    const int before = order;
    refer(o);
    const float d = far() ? (m - old.m) * kLog2e : fmaf(-old.m, kLog2e, c), e = ex2(-d);
    if (before <= kNegInf || e == 0.0f) {
      s = old.s * 0.0f;  // a NaN stays
      t = 0.0f;
    } else {
      s = e * (own && lane == 0 ? old.s + 1.0f : old.s);
      t = fmaf(e, old.t, d * s);
    }
  }
  // A logit's share of the sums. Far below the maximum (or excluded) it adds 0, not 0 * -inf.
  template <bool FAR>
  __device__ __forceinline__ void add(float x) {
    const float d = fmaxf(FAR ? (x - m) * kLog2e : fmaf(x, kLog2e, -c), -200.0f);
    const float e = ex2(d);
    s += e;
    t = fmaf(-d, e, t);
  }
};

// The largest in order of each of four blocks, for the warp; the largest of
// them. `real(u, j)`: value j of block u is the row's (`whole`: all are). nan:
// set to a NaN that a lane meets. lane_top: raised to the lane's own largest of each block.
template <class Real>
__device__ __forceinline__ int step_max(const float (&x)[kStep][4], int (&bm)[kStep], float& nan, bool whole,
                                        Real real, int* lane_top = nullptr) {
  float m[kStep], least = INFINITY;
#pragma unroll
  for (int u = 0; u < kStep; u++) {
    m[u] = x[u][0];
#pragma unroll
    for (int j = 1; j < 4; j++) asm("max.NaN.f32 %0, %0, %1;" : "+f"(m[u]) : "f"(x[u][j]));
    asm("min.NaN.f32 %0, %0, %1;" : "+f"(least) : "f"(fabsf(m[u])));
    bm[u] = order(m[u]);
  }
  // By integers where floats do not decide: NaNs, of which one sign is the
  // highest in order and the other the lowest, zeros of both signs, and
  // places behind the row's ends, which are lowest of all.
  if (!whole || !(least > 0.0f)) {
#pragma unroll
    for (int u = 0; u < kStep; u++) {
      bm[u] = INT_MIN;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        if (real(u, j)) bm[u] = max(bm[u], order(x[u][j]));
        if (isnan(x[u][j])) nan = x[u][j];
      }
    }
  }
  if (lane_top)
#pragma unroll
    for (int u = 0; u < kStep; u++) lane_top[u] = max(lane_top[u], bm[u]);
  __syncwarp();
#pragma unroll
  for (int u = 0; u < kStep; u++) bm[u] = __reduce_max_sync(0xffffffffu, bm[u]);
  return max(max(bm[0], bm[1]), max(bm[2], bm[3]));
}

// Adds a step's logits, none above a.m, to the sums. With `leave`, the first
// place of a.m in the step stays outside them.
__device__ __forceinline__ void step_add(Running& a, float (&x)[kStep][4], int lane, bool leave) {
  if (a.order <= kNegInf) return;  // nothing but excluded tokens so far
  if (leave) {
    a.own = true;
    int mine = kStep * 4;
#pragma unroll
    for (int i = kStep * 4 - 1; i >= 0; i--)
      if (x[i / 4][i % 4] == a.m) mine = i;
    const unsigned who = __ballot_sync(0xffffffffu, mine < kStep * 4);
    if (lane == __ffs(who) - 1) {
#pragma unroll
      for (int i = 0; i < kStep * 4; i++)
        if (i == mine) x[i / 4][i % 4] = -INFINITY;
    }
  }
  if (a.far()) {
    for (int i = 0; i < kStep * 4; i++) a.add<true>(x[i / 4][i % 4]);
    return;
  }
#pragma unroll
  for (int i = 0; i < kStep * 4; i++) a.add<false>(x[i / 4][i % 4]);
}

// A key with k <= #{keys >= it} <= most: bisection over 64-bit keys that no
// two entries share, none above hi and at least k of them lo or above.
// count(key) is called by all threads and is the same for all.
template <class Count>
__device__ __forceinline__ unsigned long long key_bound(int k, int most, unsigned long long lo, unsigned long long hi,
                                                        Count count) {
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
  float4* part;     // piece of row r by CTA c: [r + c]
  unsigned long long* part_best;  // its largest logit, likewise
  int* block_max;   // [rows][steps * kStep], or null
  unsigned* ticket;
  float2* peak;     // [rows] maximum and log Z for k_alternatives
  int vocab, top;
  int steps;        // of a row, whatever its alignment
  int pitch;        // of a row where they are dealt out: steps, or a multiple of run
  long long total;  // rows * pitch
  long long run;    // steps of a CTA
};

struct ScoreShared {
  Soft soft[kScoreWarps];
  int last, n_blocks, n_cand;
  int first[kScoreWarps];
  int counts[2][kScoreWarps];
  uint2 range[kScoreWarps];
  unsigned long long best[kScoreWarps];
  unsigned long long cand[kCand];
  int blocks[kPicked];
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

// A bound for the keys that the CTA's threads hold (N each, 0 for none; `held`,
// at least k, in all): between k and slack(k) keys are at or above it.
template <int N>
__device__ __forceinline__ unsigned long long own_bound(int k, const unsigned long long (&own)[N], int held, int& turn,
                                                        ScoreShared& sh) {
  if (held <= slack(k)) return 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // None is above the largest; where every thread has one, the least of the
  // threads' largest has 256 >= k at or above it.
  unsigned high = 0;
#pragma unroll
  for (int i = 0; i < N; i++) high = max(high, unsigned(own[i] >> 32));
  const unsigned low = __reduce_min_sync(0xffffffffu, high);
  high = __reduce_max_sync(0xffffffffu, high);
  if (lane == 0) sh.range[warp] = make_uint2(low, high);
  __syncthreads();
  const uint2 w = sh.range[lane % kScoreWarps];
  const unsigned long long lo = static_cast<unsigned long long>(__reduce_min_sync(0xffffffffu, w.x)) << 32;
  const unsigned long long hi =
      (static_cast<unsigned long long>(__reduce_max_sync(0xffffffffu, w.y)) << 32) | 0xFFFFFFFFull;
  return max(1ull, key_bound(k, slack(k), lo, hi, [&](unsigned long long key) {
    int c = 0;
#pragma unroll
    for (int i = 0; i < N; i++) c += own[i] >= key;
    return cta_sum(c, turn, sh);
  }));
}

// The keys of a lane's granule of block b (0 where it is not the row's).
__device__ __forceinline__ void granule_keys(const Row& r, int b, int lane, float4 v, unsigned long long (&key)[4]) {
  const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const int at = r.element(b, lane, j);
    key[j] = at >= 0 && at < r.vocab ? order_key(order(x[j]), uint32_t(at)) : 0ull;
  }
}

// Candidates among the listed blocks where too many elements pass the blocks'
// bound (neighbours that are all large, or fewer blocks than k): the same search
// among the blocks' granules, each the largest of four, leaves at most 4 slack(k).
__device__ __noinline__ void granule_candidates(const Row& r, int k, int& turn, ScoreShared& sh) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nb = sh.n_blocks;
  auto load = [&](int i, unsigned long long (&key)[4]) {
    const int b = sh.blocks[i * kScoreWarps + warp];
    granule_keys(r, b, lane, r.inside(b) ? r.load(b, lane) : r.load_end(b, lane, 0.f), key);
  };
  unsigned long long own[kGranules];
  int held = 0;
#pragma unroll
  for (int i = 0; i < kGranules; i++) {
    own[i] = 0;
    if (i * kScoreWarps + warp < nb) {
      unsigned long long key[4];
      load(i, key);
      own[i] = max(max(key[0], key[1]), max(key[2], key[3]));
      held += own[i] != 0;
    }
  }
  held = cta_sum(held, turn, sh);
  const unsigned long long bound = own_bound(min(k, held), own, held, turn, sh);
  const unsigned long long least = held < k ? 1ull : bound;
  __syncthreads();
  if (threadIdx.x == 0) sh.n_cand = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kGranules; i++) {
    if (own[i] < bound) continue;
    unsigned long long key[4];
    load(i, key);
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (key[j] >= least) sh.cand[atomicAdd(&sh.n_cand, 1)] = key[j];
  }
  __syncthreads();
}

__device__ __forceinline__ const int* row_table(const ScoreArgs& a, size_t row) {
  return a.block_max + row * size_t(a.steps) * kStep;
}
// A thread's entries of the row's table, where all of them fit the CTA's registers.
__device__ __forceinline__ void table_entries(const ScoreArgs& a, const Row& r, size_t row, int (&entry)[kOwn]) {
#pragma unroll
  for (int i = 0; i < kOwn; i++) {
    const int b = int(threadIdx.x) + i * kScoreThreads;
    entry[i] = r.blocks <= kOwn * kScoreThreads && b < r.blocks ? __ldcg(row_table(a, row) + b) : 0;
  }
}

// The `top` largest of a row with maximum m, ranked: by the whole CTA, whose
// table_entries() are there.
__device__ __forceinline__ void alternatives(const ScoreArgs& a, const Row& r, size_t row, float m, float logz,
                                             const int (&entry)[kOwn], ScoreShared& sh) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int k = a.top;
  const int* block_max = row_table(a, row);
  int turn = 0;
  if (threadIdx.x == 0) sh.n_blocks = sh.n_cand = 0;
  // The blocks with the largest maxima: k of them, or more where that ends the search sooner.
  auto block_key = [&](int b) { return order_key(__ldcg(block_max + b), uint32_t(b)); };
  const int kb = min(k, r.blocks);
  unsigned long long bound;
  if (r.blocks <= kOwn * kScoreThreads) {
    unsigned long long own[kOwn];
#pragma unroll
    for (int i = 0; i < kOwn; i++) {
      const int b = int(threadIdx.x) + i * kScoreThreads;
      own[i] = b < r.blocks ? order_key(entry[i], uint32_t(b)) : 0ull;
    }
    bound = own_bound(kb, own, r.blocks, turn, sh);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kOwn; i++)
      if (own[i] >= bound) sh.blocks[atomicAdd(&sh.n_blocks, 1)] = int(threadIdx.x) + i * kScoreThreads;
  } else {
    bound = key_bound(k, slack(k), 0ull, ~0ull, [&](unsigned long long key) {
      int c = 0;
      for (int b = threadIdx.x; b < r.blocks; b += kScoreThreads) c += block_key(b) >= key;
      return cta_sum(c, turn, sh);
    });
    __syncthreads();
    for (int b = threadIdx.x; b < r.blocks; b += kScoreThreads)
      if (block_key(b) >= bound) sh.blocks[atomicAdd(&sh.n_blocks, 1)] = b;
  }
  __syncthreads();
  const int nb = sh.n_blocks;
  // Candidates: the elements at least as large as the smallest of the picked maxima (k of these exist).
  const bool all = r.blocks <= slack(kb);  // no bound was needed
  if (!all) {
    const unsigned long long least = bound & 0xFFFFFFFF00000000ull;
    constexpr int kBatch = 4;
    for (int i0 = warp; i0 < nb; i0 += kBatch * kScoreWarps) {
      float4 v[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; i++)
        if (i0 + i * kScoreWarps < nb) {
          const int b = sh.blocks[i0 + i * kScoreWarps];
          v[i] = r.inside(b) ? r.load(b, lane) : r.load_end(b, lane, 0.f);
        }
#pragma unroll
      for (int i = 0; i < kBatch; i++)
        if (i0 + i * kScoreWarps < nb) {
          unsigned long long key[4];
          granule_keys(r, sh.blocks[i0 + i * kScoreWarps], lane, v[i], key);
#pragma unroll
          for (int j = 0; j < 4; j++)
            if (key[j] >= least && key[j]) {
              const int at = atomicAdd(&sh.n_cand, 1);
              if (at < kCand) sh.cand[at] = key[j];
            }
        }
    }
    __syncthreads();
  }
  if (all || sh.n_cand > kCand) granule_candidates(r, k, turn, sh);
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

// The sets of `n` lanes joined, on every lane: lane pairs join the lower
// lane's set first on both sides, so that all get the same bits.
__device__ __forceinline__ Soft soft_lanes(Soft p, int n, int lane) {
  for (int o = 1; o < n; o <<= 1) {
    const Soft q{__shfl_xor_sync(0xffffffffu, p.m, o), __shfl_xor_sync(0xffffffffu, p.s, o),
                 __shfl_xor_sync(0xffffffffu, p.t, o), __shfl_xor_sync(0xffffffffu, p.own, o)};
    p = (lane & o) ? soft_join(q, p) : soft_join(p, q);
  }
  return p;
}
// The sets of the CTA's warps (the same on each warp's lanes) joined, on every thread.
__device__ __forceinline__ Soft soft_cta(const Soft& p, int warp, int lane, ScoreShared& sh) {
  if (lane == 0) sh.soft[warp] = p;
  __syncthreads();
  return soft_lanes(sh.soft[lane % kScoreWarps], kScoreWarps, lane);
}

// What a call does about the alternatives: nothing, or what k_alternatives needs
// (the table and a.peak, where a.block_max is given); the one most likely token, which
// is the place of the maximum and needs no table; several, by the CTA that
// finishes a row.
enum ScoreTop { kTopApart, kTopOne, kTopMany };
template <int TOP>
__global__ void __launch_bounds__(kScoreThreads, 4) k_score(ScoreArgs a) {
  __shared__ ScoreShared sh;
  pdl_launch_dependents();
  pdl_wait();
  a.logits = after_wait(a.logits);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float nan = __int_as_float(0x7FC00000);
  long long g = blockIdx.x * a.run;
  const long long g1 = min(a.total, g + a.run);
  while (g < g1) {
    const size_t row = size_t(g / a.pitch);
    const int s0 = int(g - (long long)row * a.pitch), end = int(min((long long)a.pitch, s0 + (g1 - g)));
    const int s1 = min(end, a.steps);
    g += end - s0;
    const Row r(a.logits, row, a.vocab);
    int* block_max = TOP != kTopOne && a.block_max ? a.block_max + row * size_t(a.steps) * kStep : nullptr;
    // The token's logit, for whoever finishes the row: on its way while the others are read.
    float given = nan;
    if (threadIdx.x == 0) {
      const uint32_t tok = a.tokens[row];
      if (tok < uint32_t(a.vocab)) given = ld_f32(r.base + r.shift + tok);
    }
    int st = s0 + warp;
    bool whole = false;
    float x[kStep][4], met = 0.f;
    int bm[kStep], top = INT_MIN;
    unsigned long long best = 0;  // kTopOne: the largest logit, if this warp met it
    auto load = [&] {
      const int b = st * kStep;
      whole = r.inside(b) && r.inside(b + kStep - 1);
#pragma unroll
      for (int u = 0; u < kStep; u++) {
        const float4 v = whole ? r.load(b + u, lane) : r.load_end(b + u, lane, -INFINITY);
        x[u][0] = v.x, x[u][1] = v.y, x[u][2] = v.z, x[u][3] = v.w;
      }
      top = step_max(x, bm, met, whole, [&](int u, int j) {
        const int at = r.element(b + u, lane, j);
        return whole || (at >= 0 && at < a.vocab);
      });
      if (block_max && lane == 0) reinterpret_cast<int4*>(block_max)[st] = make_int4(bm[0], bm[1], bm[2], bm[3]);
    };
    // kTopOne: the step's largest is larger than all before it; its first place.
    auto keep = [&] {
      unsigned at = 0xFFFFFFFFu;
#pragma unroll
      for (int i = kStep * 4 - 1; i >= 0; i--) {
        const int e = r.element(st * kStep + i / 4, lane, i % 4);
        if (order(x[i / 4][i % 4]) == top && e >= 0 && e < a.vocab) at = unsigned(e);
      }
      best = order_key(top, __reduce_min_sync(0xffffffffu, at));
    };
    if (st < s1) load();
    if (lane == 0) sh.first[warp] = top;
    __syncthreads();
    int common = sh.first[lane % kScoreWarps];
    const unsigned holders = __ballot_sync(0xffffffffu, common == __reduce_max_sync(0xffffffffu, common));
    common = __shfl_sync(0xffffffffu, common, __ffs(holders) - 1);
    Running run(max(common, kNegInf));
    if (st < s1) {
      const bool holder = warp == __ffs(holders) - 1;
      if (TOP == kTopOne && holder) keep();
      step_add(run, x, lane, holder);
      for (st += kScoreWarps; st < s1; st += kScoreWarps) {
        load();
        const bool higher = top > run.order;
        if (higher) {
          run.raise(top, lane);
          if (TOP == kTopOne) keep();
        }
        step_add(run, x, lane, higher);
      }
    }
    run.s += met * 0.0f;  // a NaN stays
    Soft s = run.settled();
    s.s = warp_sum(s.s);
    s.t = warp_sum(s.t);
    if (TOP == kTopOne && lane == 0) sh.best[warp] = best;
    s = soft_cta(s, warp, lane, sh);
    if (TOP == kTopOne) best = warp_umax64(sh.best[lane % kScoreWarps]);
    // Pieces of this row: those of the CTAs whose runs meet it.
    int entry[kOwn];
    const long long c0 = (long long)row * a.pitch / a.run, c1 = ((long long)(row + 1) * a.pitch - 1) / a.run;
    if (c1 > c0) {
      if (threadIdx.x == 0) {
        a.part[row + blockIdx.x] = make_float4(s.m, s.s, s.t, s.own);
        if (TOP == kTopOne) a.part_best[row + blockIdx.x] = best;
        unsigned before;  // releases this CTA's writes, acquires those of the CTAs before it
        asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(before) : "l"(a.ticket + row) : "memory");
        sh.last = before == unsigned(c1 - c0);
      }
      __syncthreads();
      if (!sh.last) {
        __syncthreads();  // sh.last is read before the next piece writes it
        continue;
      }
      // On their way while the sums are joined.
      if (TOP == kTopMany) table_entries(a, r, row, entry);
      Soft p{-INFINITY, 0.f, 0.f, 0.f};
      for (long long c = c0 + threadIdx.x; c <= c1; c += kScoreThreads) {
        const float4 q = __ldcg(a.part + row + c);
        p = soft_join(p, Soft{q.x, q.y, q.z, q.w});
        if (TOP == kTopOne) best = max(best, __ldcg(a.part_best + row + c));
      }
      if (TOP == kTopOne) {
        best = warp_umax64(best);
        if (lane == 0) sh.best[warp] = best;
      }
      s = soft_cta(soft_lanes(p, 32, lane), warp, lane, sh);
      if (TOP == kTopOne) best = warp_umax64(sh.best[lane % kScoreWarps]);
      if (threadIdx.x == 0) a.ticket[row] = 0;
    } else if (TOP == kTopMany) {
      table_entries(a, r, row, entry);
    }
    const bool bad = !(s.m < INFINITY) || s.m == -INFINITY || isnan(s.s);
    const float logz = bad ? nan : log1pf(s.s);
    if (threadIdx.x == 0) {
      a.entropy[row] = logz + kLn2 * s.t / (1.0f + s.s);
      a.logprob[row] = (given - s.m) - logz;
      if (TOP == kTopOne) {
        a.top_ids[row] = argmax_index(best);
        a.top_logprobs[row] = (unorder(int(uint32_t(best >> 32) ^ 0x80000000u)) - s.m) - logz;
      } else if (TOP == kTopApart && a.block_max) {
        a.peak[row] = make_float2(s.m, logz);
      }
    }
    if constexpr (TOP == kTopMany) alternatives(a, r, row, s.m, logz, entry, sh);
    __syncthreads();  // shared memory is free for the next piece
  }
}

// The alternatives of row blockIdx.x.
__global__ void __launch_bounds__(kScoreThreads, 4) k_alternatives(ScoreArgs a) {
  __shared__ ScoreShared sh;
  pdl_launch_dependents();
  pdl_wait();
  a.logits = after_wait(a.logits);
  const size_t row = blockIdx.x;
  const Row r(a.logits, row, a.vocab);
  int entry[kOwn];
  table_entries(a, r, row, entry);
  const float2 p = a.peak[row];
  alternatives(a, r, row, p.x, p.y, entry, sh);
}

// Short rows, of at most S steps: a warp each, the whole row in its registers; no
// pieces, no barriers. A few alternatives are the largest remaining logit, time
// after time; more are those above a bound, ranked (1400 x 500: 8 us with five, 10
// with twenty, which took 19 one by one; by CTAs 36).
template <int S>
__global__ void __launch_bounds__(kScoreThreads) k_score_rows(ScoreArgs a, int rows) {
  pdl_launch_dependents();
  pdl_wait();
  a.logits = after_wait(a.logits);
  const int lane = threadIdx.x & 31;
  const long long row = (long long)blockIdx.x * kScoreWarps + (threadIdx.x >> 5);
  if (row >= rows) return;
  const Row r(a.logits, size_t(row), a.vocab);
  const float nan = __int_as_float(0x7FC00000);
  const uint32_t tok = a.tokens[row];
  const float given = tok < uint32_t(a.vocab) ? ld_f32(r.base + r.shift + tok) : nan;
  float x[S][kStep][4], met = 0.f;
  int top[S], common = INT_MIN;
#pragma unroll
  for (int s = 0; s < S; s++)
#pragma unroll
    for (int u = 0; u < kStep; u++) {
      const int b = s * kStep + u;
      const float4 v = r.inside(b) ? r.load(b, lane) : r.load_end(b, lane, -INFINITY);
      x[s][u][0] = v.x, x[s][u][1] = v.y, x[s][u][2] = v.z, x[s][u][3] = v.w;
    }
  auto real = [&](int s, int i) {
    const int at = r.element(s * kStep + i / 4, lane, i % 4);
    return at >= 0 && at < a.vocab;
  };
#pragma unroll
  for (int s = 0; s < S; s++) {
    int bm[kStep];
    const bool whole = r.inside(s * kStep) && r.inside(s * kStep + kStep - 1);
    top[s] = step_max(x[s], bm, met, whole, [&](int u, int j) { return whole || real(s, 4 * u + j); });
    common = max(common, top[s]);
  }
  // The logits in order; what is not the row's is out from the start.
  int o[S][kStep * 4];
  unsigned gone[S];
  if (a.top) {
#pragma unroll
    for (int s = 0; s < S; s++) {
      gone[s] = 0;
#pragma unroll
      for (int i = 0; i < kStep * 4; i++) {
        o[s][i] = order(x[s][i / 4][i % 4]);
        gone[s] |= unsigned(!real(s, i)) << i;
      }
    }
  }
  Running run(max(common, kNegInf));
  bool leave = true;
#pragma unroll
  for (int s = 0; s < S; s++) {
    const bool here = leave && top[s] == common;
    step_add(run, x[s], lane, here);
    leave = leave && !here;
  }
  run.s += met * 0.0f;  // a NaN stays
  Soft f = run.settled();
  f.s = warp_sum(f.s);
  f.t = warp_sum(f.t);
  const bool bad = !(f.m < INFINITY) || f.m == -INFINITY || isnan(f.s);
  const float logz = bad ? nan : log1pf(f.s);
  if (lane == 0) {
    a.entropy[row] = logz + kLn2 * f.t / (1.0f + f.s);
    a.logprob[row] = (given - f.m) - logz;
  }
  // A lane's largest remaining logit: its order and its first place.
  bool have = false;
  int best = 0, place = 0;
  auto largest = [&] {
    have = false;
#pragma unroll
    for (int s = 0; s < S; s++)
#pragma unroll
      for (int i = 0; i < kStep * 4; i++)
        if (!((gone[s] >> i) & 1) && (!have || o[s][i] > best)) have = true, best = o[s][i], place = s * kStep * 4 + i;
  };
  if (a.top) largest();
  if (a.top > kOneByOne) {
    auto each = [&](auto f) {
#pragma unroll
      for (int s = 0; s < S; s++)
#pragma unroll
        for (int i = 0; i < kStep * 4; i++)
          f(!((gone[s] >> i) & 1) ? order_key(o[s][i], uint32_t(r.element(s * kStep + i / 4, lane, i % 4))) : 0ull);
    };
    // None is above the largest; the lanes' largest are 32 keys at or above their least.
    const unsigned mine = have ? unsigned(best) ^ 0x80000000u : 0u;
    const unsigned low = __reduce_min_sync(0xffffffffu, mine), high = __reduce_max_sync(0xffffffffu, mine);
    const unsigned long long lo = a.top <= 32 ? static_cast<unsigned long long>(low) << 32 : 0ull;
    const unsigned long long hi = (static_cast<unsigned long long>(high) << 32) | 0xFFFFFFFFull;
    const unsigned long long bound = max(1ull, key_bound(a.top, slack(a.top), lo, hi, [&](unsigned long long key) {
      int c = 0;
      each([&](unsigned long long k) { c += k >= key; });
      return __reduce_add_sync(0xffffffffu, c);
    }));
    __shared__ unsigned long long rooms[kScoreWarps][kPicked];
    unsigned long long* room = rooms[threadIdx.x >> 5];
    int n = 0;
    each([&](unsigned long long k) {
      const unsigned who = __ballot_sync(0xffffffffu, k >= bound);
      if (k >= bound) room[n + __popc(who & ((1u << lane) - 1))] = k;
      n += __popc(who);
    });
    __syncwarp();
    for (int i = lane; i < n; i += 32) {
      const unsigned long long k = room[i];
      int rank = 0;
      for (int j = 0; j < n; j++) rank += room[j] > k;
      if (rank < a.top) {
        a.top_ids[row * a.top + rank] = argmax_index(k);
        a.top_logprobs[row * a.top + rank] = (unorder(int(uint32_t(k >> 32) ^ 0x80000000u)) - f.m) - logz;
      }
    }
    return;
  }
  for (int k = 0; k < a.top; k++) {
    // Of the lanes with the warp's largest, the one whose element comes first.
    const int m = __reduce_max_sync(0xffffffffu, have ? best : INT_MIN);
    const int e = r.element(place / 4, lane, place % 4);
    const int first = __reduce_min_sync(0xffffffffu, have && best == m ? e : INT_MAX);
    if (have && e == first) {
      a.top_ids[row * a.top + k] = uint32_t(e);
      a.top_logprobs[row * a.top + k] = (unorder(m) - f.m) - logz;
#pragma unroll
      for (int s = 0; s < S; s++)
        if (place / (kStep * 4) == s) gone[s] |= 1u << (place % (kStep * 4));
      largest();
    }
    __syncwarp();
  }
}

// Rows of up to kRowSteps steps where there are enough of them: a warp each again,
// which goes through its row and has the next step on its way meanwhile. For
// the alternatives the row falls into 128 sets, each lane's places in the four
// blocks of every step: k of the sets' largest logits are at least the k-th of
// them, which bounds the k-th logit from below closely (about 1.4 k logits reach it at
// k = 64). The blocks that reach it, by their maxima, are read again. 2048 x 5000, us,
// no and twenty alternatives: 10.2 and 19.7, by k_score and k_alternatives 17.2 and 48.1 (from memory 11.5 and 21.0).
constexpr int kRowSteps = 64;
constexpr int kRowWarps = 4;
constexpr int kRoom = 256;  // candidates that a warp holds
static_assert(kRoom >= kPicked + kBlock, "after a cut there is room for a block");
__global__ void __launch_bounds__(32 * kRowWarps) k_score_long_rows(ScoreArgs a, int rows) {
  __shared__ int4 tables[kRowWarps][kRowSteps];
  __shared__ unsigned long long rooms[kRowWarps][kRoom];
  pdl_launch_dependents();
  pdl_wait();
  a.logits = after_wait(a.logits);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long row = (long long)blockIdx.x * kRowWarps + warp;
  if (row >= rows) return;
  const Row r(a.logits, size_t(row), a.vocab);
  const float nan = __int_as_float(0x7FC00000);
  const uint32_t tok = a.tokens[row];
  const float given = tok < uint32_t(a.vocab) ? ld_f32(r.base + r.shift + tok) : nan;
  auto whole = [&](int st) { return r.inside(st * kStep) && r.inside(st * kStep + kStep - 1); };
  auto fetch = [&](int st, float4 (&v)[kStep]) {
    const bool w = whole(st);
#pragma unroll
    for (int u = 0; u < kStep; u++) {
      const int b = st * kStep + u;
      v[u] = w ? r.load(b, lane) : r.load_end(b, lane, -INFINITY);
    }
  };
  float met = 0.f;
  int sets[kStep] = {INT_MIN, INT_MIN, INT_MIN, INT_MIN};
  Running run(kNegInf);
  float4 next[kStep];
  fetch(0, next);
#pragma unroll 2
  for (int st = 0; st < a.steps; st++) {
    float x[kStep][4];
#pragma unroll
    for (int u = 0; u < kStep; u++) x[u][0] = next[u].x, x[u][1] = next[u].y, x[u][2] = next[u].z, x[u][3] = next[u].w;
    if (st + 1 < a.steps) fetch(st + 1, next);
    int bm[kStep];
    const bool w = whole(st);
    const int top = step_max(x, bm, met, w, [&](int u, int j) {
      const int at = r.element(st * kStep + u, lane, j);
      return w || (at >= 0 && at < a.vocab);
    }, sets);
    if (lane == 0) tables[warp][st] = make_int4(bm[0], bm[1], bm[2], bm[3]);
    const bool higher = top > run.order;
    if (higher) run.raise(top, lane);
    step_add(run, x, lane, higher);
  }
  run.s += met * 0.0f;  // a NaN stays
  Soft f = run.settled();
  f.s = warp_sum(f.s);
  f.t = warp_sum(f.t);
  const bool bad = !(f.m < INFINITY) || f.m == -INFINITY || isnan(f.s);
  const float logz = bad ? nan : log1pf(f.s);
  if (lane == 0) {
    a.entropy[row] = logz + kLn2 * f.t / (1.0f + f.s);
    a.logprob[row] = (given - f.m) - logz;
  }
  const int k = a.top;
  if (!k) return;
  // From here on no key below `least` is among the k largest.
  unsigned long long least;
  unsigned own[kStep], hi;
  {
#pragma unroll
    for (int u = 0; u < kStep; u++) own[u] = unsigned(sets[u]) ^ 0x80000000u;
    const unsigned high = max(max(own[0], own[1]), max(own[2], own[3]));
    hi = __reduce_max_sync(0xffffffffu, high);
    unsigned lo = hi;
    if (k > 1) {
      lo = __reduce_min_sync(0xffffffffu, k <= 32 ? high : min(min(own[0], own[1]), min(own[2], own[3])));
      for (unsigned top = hi; lo < top;) {  // lo: reached by k sets at least
        const unsigned mid = lo + (top - lo) / 2 + 1;
        const int c =
            __reduce_add_sync(0xffffffffu, (own[0] >= mid) + (own[1] >= mid) + (own[2] >= mid) + (own[3] >= mid));
        if (c >= k) {
          lo = mid;
          if (c <= k + k / 8) break;
        } else {
          top = mid - 1;
        }
      }
    }
    least = max(1ull, static_cast<unsigned long long>(lo) << 32);
  }
  const unsigned long long most = (static_cast<unsigned long long>(hi) << 32) | 0xFFFFFFFFull;
  unsigned long long* room = rooms[warp];
  int n = 0;
  // Cuts the candidates down to slack(k), where rows rise or have many equal logits.
  auto cut = [&] {
    unsigned long long mine[kRoom / 32];
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kRoom / 32; i++) mine[i] = i * 32 + lane < n ? room[i * 32 + lane] : 0ull;
    least = key_bound(k, slack(k), least, most, [&](unsigned long long key) {
      int c = 0;
#pragma unroll
      for (int i = 0; i < kRoom / 32; i++) c += mine[i] >= key;
      return __reduce_add_sync(0xffffffffu, c);
    });
    __syncwarp();
    n = 0;
#pragma unroll
    for (int i = 0; i < kRoom / 32; i++) {
      const unsigned who = __ballot_sync(0xffffffffu, mine[i] >= least);
      if (mine[i] >= least) room[n + __popc(who & ((1u << lane) - 1))] = mine[i];
      n += __popc(who);
    }
  };
  const int* table = reinterpret_cast<const int*>(tables[warp]);
  __syncwarp();
  for (int b0 = 0; b0 < r.blocks; b0 += 32) {
    const int b = b0 + lane;
    unsigned picked = __ballot_sync(0xffffffffu, b < r.blocks && order_key(table[min(b, r.blocks - 1)], 0) >= least);
    while (picked) {
      constexpr int kBatch = 4;
      float4 v[kBatch];
      int bs[kBatch], m = 0;
#pragma unroll
      for (int i = 0; i < kBatch; i++) {
        if (!picked) break;
        bs[i] = b0 + __ffs(picked) - 1;
        picked &= picked - 1;
        v[i] = r.inside(bs[i]) ? r.load(bs[i], lane) : r.load_end(bs[i], lane, 0.f);
        m = i + 1;
      }
#pragma unroll
      for (int i = 0; i < kBatch; i++) {
        if (i >= m) break;
        if (n + kBlock > kRoom) cut();
        const float x[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const int o = order(x[j]);
          if (!__any_sync(0xffffffffu, (unsigned(o) ^ 0x80000000u) >= unsigned(least >> 32))) continue;
          const int at = r.element(bs[i], lane, j);
          const unsigned long long key = at >= 0 && at < r.vocab ? order_key(o, uint32_t(at)) : 0ull;
          const unsigned who = __ballot_sync(0xffffffffu, key >= least);
          if (key >= least) room[n + __popc(who & ((1u << lane) - 1))] = key;
          n += __popc(who);
        }
      }
    }
  }
  if (n > kPicked) cut();
  __syncwarp();
  // Each candidate's rank: a lane's up to four at once, against all.
  constexpr int kMine = (kPicked + 31) / 32;
  unsigned long long mine[kMine];
  int rank[kMine];
#pragma unroll
  for (int i = 0; i < kMine; i++) mine[i] = i * 32 + lane < n ? room[i * 32 + lane] : 0ull, rank[i] = 0;
  for (int j = 0; j < n; j++) {
    const unsigned long long other = room[j];
#pragma unroll
    for (int i = 0; i < kMine; i++)
      if (i * 32 < n) rank[i] += other > mine[i];
  }
#pragma unroll
  for (int i = 0; i < kMine; i++)
    if (mine[i] && rank[i] < k) {
      a.top_ids[row * k + rank[i]] = argmax_index(mine[i]);
      a.top_logprobs[row * k + rank[i]] = (unorder(int(uint32_t(mine[i] >> 32) ^ 0x80000000u)) - f.m) - logz;
    }
}

// Steps of a row, whatever its alignment.
int score_steps(size_t vocab) { return int((vocab + 3 + kStep * kBlock - 1) / (kStep * kBlock)); }

// How k_score's CTAs share the rows: a row each; each row cut into equal pieces, a
// CTA for each; or all rows' steps in equal runs for the CTAs that run at once. By the steps
// of the CTA that has most, a join counted as 32 and two pieces for a CTA as 64 (us, without alternatives:
// 1 x 5000 4.1 whole and 5.1 cut, 1 x 32000 7.1 and 5.5; 64 x 32000 7.8 whole, 11.4 in equal runs,
// 7.2 in pieces; 2048 x 32000 51.9 whole and 55.3 in runs).
void deal(ScoreArgs& a, long long n, long long ctas) {
  const long long whole = (n + ctas - 1) / ctas * a.steps;
  const long long even = std::max<long long>((n * a.steps + ctas - 1) / ctas, std::min(a.steps, kScoreWarps));
  const long long each = std::max<long long>(1, ctas / n);  // pieces of a row
  const long long piece = std::max<long long>((a.steps + each - 1) / each, std::min(a.steps, kScoreWarps));
  a.run = a.pitch = a.steps;
  long long least = whole;
  if (piece < a.steps && piece + 32 < least) {
    least = piece + 32;
    a.run = piece;
    a.pitch = int((a.steps + piece - 1) / piece * piece);
  }
  if (even + 64 < least) a.run = even, a.pitch = a.steps;
  a.total = n * a.pitch;
}

}  // namespace
}  // namespace tb

namespace {

// Whether p is device (or managed) memory, and whose. By the driver's query of
// just these two attributes, a microsecond less than the runtime's of all of them.
int where_is(const void* p, bool* on_device, int* ordinal) {
  static PFN_cuPointerGetAttributes_v7000 query = [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult r{};
    if (cudaGetDriverEntryPoint("cuPointerGetAttributes", &fn, cudaEnableDefault, &r) != cudaSuccess ||
        r != cudaDriverEntryPointSuccess)
      fn = nullptr;
    return reinterpret_cast<PFN_cuPointerGetAttributes_v7000>(fn);
  }();
  if (!query) return rt::fail(TB200_ERR_CUDA, "cuPointerGetAttributes is not available from the driver");
  CUmemorytype type = CUmemorytype(0);  // stays so for memory that CUDA does not know
  CUpointer_attribute what[2] = {CU_POINTER_ATTRIBUTE_MEMORY_TYPE, CU_POINTER_ATTRIBUTE_DEVICE_ORDINAL};
  void* to[2] = {&type, ordinal};
  const CUresult r = query(2, what, to, CUdeviceptr(reinterpret_cast<uintptr_t>(p)));
  if (r != CUDA_SUCCESS)
    return rt::fail(TB200_ERR_CUDA, "score: cuPointerGetAttributes failed (" + std::to_string(int(r)) + ")");
  *on_device = type == CU_MEMORYTYPE_DEVICE || type == CU_MEMORYTYPE_UNIFIED;
  return TB200_OK;
}

}  // namespace

extern "C" {

int tb200_scorer_new(tb200_device* dev, size_t rows, size_t vocab, size_t top, tb200_scorer** out) {
  ARG_CHECK(dev && out, "null argument");
  ARG_CHECK(rows >= 1 && rows <= (size_t(1) << 24), "bad number of rows");
  ARG_CHECK(vocab >= 1 && vocab <= (size_t(1) << 30), "bad vocabulary");
  ARG_CHECK(top <= size_t(tb::kScoreMaxTop) && top <= vocab, "top must be at most 64 and the vocabulary");
  if (int rc = rt::use(dev)) return rc;
  auto* s = new tb200_scorer;
  s->dev = dev;
  s->rows = rows;
  s->vocab = vocab;
  s->top = int(top);
  const size_t blocks = size_t(tb::score_steps(vocab)) * tb::kStep;
  int per_sm = 0;
  cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, tb::k_score<tb::kTopMany>, tb::kScoreThreads, 0);
  s->ctas = std::max(1, per_sm) * dev->sms;
  const size_t parts = rows + size_t(s->ctas);
  if (e == cudaSuccess) e = cudaMalloc(&s->logprob, rows * 4);
  if (e == cudaSuccess) e = cudaMalloc(&s->entropy, rows * 4);
  if (e == cudaSuccess) e = cudaMalloc(&s->tokens, rows * 4);
  if (e == cudaSuccess && top) e = cudaMalloc(&s->top_ids, rows * top * 4);
  if (e == cudaSuccess && top) e = cudaMalloc(&s->top_logprobs, rows * top * 4);
  if (e == cudaSuccess) e = cudaMalloc(&s->part, parts * sizeof(float4));
  if (e == cudaSuccess) e = cudaMalloc(&s->ticket, rows * 4);
  if (e == cudaSuccess) e = cudaMemsetAsync(s->ticket, 0, rows * 4, dev->stream);
  if (e == cudaSuccess && top == 1) e = cudaMalloc(&s->part_best, parts * 8);
  if (e == cudaSuccess && top > 1) e = cudaMalloc(&s->block_max, rows * blocks * 4);
  if (e == cudaSuccess && top > 1) e = cudaMalloc(&s->peak, rows * sizeof(float2));
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
  cudaFree(s->part_best);
  cudaFree(s->block_max);
  cudaFree(s->peak);
  cudaFree(s->ticket);
  delete s;
  return TB200_OK;
}

int tb200_score_enqueue(tb200_scorer* s, const tb200_buffer* logits, const uint32_t* tokens, size_t n) {
  ARG_CHECK(s && logits && (tokens || !n), "null argument");
  ARG_CHECK(rt::of(s->dev, logits), "score: the logits were made on another device than the scorer");
  ARG_CHECK(n <= s->rows, "score: a scorer of " + std::to_string(s->rows) + " rows can't hold " + std::to_string(n));
  ARG_CHECK(logits->len >= n * s->vocab, "score: the logits buffer holds fewer than rows x vocabulary values");
  if (int rc = rt::use(s->dev)) return rc;
  if (!n) return TB200_OK;
  cudaStream_t st = s->dev->stream;
  bool on_device = false;
  int ordinal = 0;
  if (int rc = where_is(tokens, &on_device, &ordinal)) return rc;
  if (on_device) {
    ARG_CHECK(ordinal == s->dev->ordinal, "score: the tokens are in another device's memory");
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
  a.steps = tb::score_steps(s->vocab);
  tb::deal(a, (long long)n, s->ctas);
  a.part_best = s->part_best;
  a.peak = s->peak;
  const dim3 grid(unsigned((a.total + a.run - 1) / a.run)), block(tb::kScoreThreads);
  if (a.steps <= 4) {
    const dim3 warps(unsigned((n + tb::kScoreWarps - 1) / tb::kScoreWarps));
    if (a.steps == 1)
      tb::launch_pdl(tb::k_score_rows<1>, warps, block, 0, st, a, int(n));
    else if (a.steps == 2)
      tb::launch_pdl(tb::k_score_rows<2>, warps, block, 0, st, a, int(n));
    else
      tb::launch_pdl(tb::k_score_rows<4>, warps, block, 0, st, a, int(n));
  } else if (a.steps <= tb::kRowSteps && n > size_t(s->top > 1 ? 25 : 64) * a.steps) {
    // Enough rows that warps which go through theirs alone fill the GPU (us there and with a CTA a row: no
    // alternatives, 800 x 2100 5.8 and 6.5, 256 x 2100 4.6 and 4.2, 800 x 16000 21 and 12.5; five, 256 x 5000 9.6
    // and 12.5, 2048 x 32000 63 and 78, 800 x 32000 49 and 37).
    tb::launch_pdl(tb::k_score_long_rows, dim3(unsigned((n + tb::kRowWarps - 1) / tb::kRowWarps)),
                   dim3(32 * tb::kRowWarps), 0, st, a, int(n));
  } else if (s->top == 1) {
    tb::launch_pdl(tb::k_score<tb::kTopOne>, grid, block, 0, st, a);
  } else if (s->top && 2 * n <= size_t(s->ctas)) {
    tb::launch_pdl(tb::k_score<tb::kTopMany>, grid, block, 0, st, a);
  } else {
    // More rows than half the CTAs: some would find alternatives while others wait for the rest of their run.
    tb::launch_pdl(tb::k_score<tb::kTopApart>, grid, block, 0, st, a);
    if (s->top) tb::launch_pdl(tb::k_alternatives, dim3(unsigned(n)), block, 0, st, a);
  }
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
