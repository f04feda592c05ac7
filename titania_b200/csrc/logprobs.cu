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
// One launch, one pass over the logits, bound by reading them. The rows' steps
// of 512 logits, one after another, are dealt out to the CTAs in equal runs
// (whatever the number of rows, no SM waits for another's last row); a CTA's
// part of a row is a piece. A warp takes a step at a time, as four blocks of
// 128: their largest, a redux each, are both the running maximum that the sums
// refer to, so that rescaling is a rare warp-uniform branch, and the blocks'
// entries in a table of 1/128 of the logits' size. Per logit that leaves five
// instructions for the sums and one for the maximum; at ten it was bound by
// them (1111 x 151936: 142 us, against 105 us for the bytes). The CTA that finishes a row's last piece joins the pieces'
// sums, in their order, and finds the alternatives: the k largest logits lie in
// the k blocks with the largest maxima (each of those has an element at least as
// large as any element of another block), so only those blocks are read again.
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
  int* block_max = nullptr;     // [rows][a row's blocks], when there are alternatives
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
constexpr int kCand = 2048;        // candidates held in shared memory
constexpr int kOwn = 8;            // table entries or candidates a thread keeps in registers
static_assert(kCand == kOwn * kScoreThreads, "a thread's candidates fit its registers");
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

// A warp's set while it grows: m is the warp's, s and t each lane's shares of
// the sums, taken at c = f32(m log2 e) in the place of m log2 e, which saves an
// instruction a logit: what that leaves out (lo) is put right in settled().
struct Running {
  float m, c, lo, s, t;
  int order;  // of m
  __device__ __forceinline__ Running() : m(-INFINITY), c(0.f), lo(0.f), s(0.f), t(0.f), order(kNegInf) {}
  __device__ __forceinline__ Soft settled() const {
    const float f = ex2(-lo);
    return Soft{m, s * f, fmaf(lo, s, t) * f};
  }
  // Refers the sums to a larger maximum; lane 0 takes the old one's own term.
  __device__ __forceinline__ void raise(int bm, int lane) {
    const Soft old = settled();
    const float nm = unorder(bm);
    if (order > kNegInf) {
      const float d = (nm - old.m) * kLog2e, e = ex2(-d);
      if (e == 0.0f) {
        s = old.s * 0.0f;  // a NaN stays
        t = 0.0f;
      } else {
        s = lane == 0 ? fmaf(e, old.s, e) : e * old.s;
        t = fmaf(e, old.t, d * s);
      }
    }
    m = nm;
    order = bm;
    c = m * kLog2e;
    lo = huge() ? 0.f : fmaf(m, kLog2e, -c);
  }
  // Whether m log2 e may be past f32's range.
  __device__ __forceinline__ bool huge() const { return fabsf(m) > 1e38f; }
  // A logit's share of the sums. Far below the maximum (or excluded) it adds 0, not 0 * -inf.
  template <bool HUGE>
  __device__ __forceinline__ void add(float x) {
    const float d = fmaxf(HUGE ? (x - m) * kLog2e : fmaf(x, kLog2e, -c), -200.0f);
    const float e = ex2(d);
    s += e;
    t = fmaf(-d, e, t);
  }
};

// Four blocks: their largest in order go to bm, their sums to a. `real(u, j)`
// is whether value j of block u is the row's (`whole`: all are).
template <class Real>
__device__ __forceinline__ void add_step(Running& a, float4 (&v)[kStep], int (&bm)[kStep], int lane, bool whole,
                                         Real real) {
  float x[kStep][4];
  float m[kStep], least = INFINITY;
#pragma unroll
  for (int u = 0; u < kStep; u++) {
    x[u][0] = v[u].x, x[u][1] = v[u].y, x[u][2] = v[u].z, x[u][3] = v[u].w;
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
        if (isnan(x[u][j])) a.s = x[u][j];
      }
    }
  }
  __syncwarp();
#pragma unroll
  for (int u = 0; u < kStep; u++) bm[u] = __reduce_max_sync(0xffffffffu, bm[u]);
  const int top = max(max(bm[0], bm[1]), max(bm[2], bm[3]));
  if (top > a.order) {  // a new maximum, the same for the warp
    a.raise(top, lane);
    // It stays out of the sums itself: its first place in the step.
    int mine = kStep * 4;
#pragma unroll
    for (int i = kStep * 4 - 1; i >= 0; i--)
      if (order(x[i / 4][i % 4]) == top && real(i / 4, i % 4)) mine = i;
    const unsigned who = __ballot_sync(0xffffffffu, mine < kStep * 4);
    if (lane == __ffs(who) - 1) {
#pragma unroll
      for (int i = 0; i < kStep * 4; i++)
        if (i == mine) x[i / 4][i % 4] = -INFINITY;
    }
  }
  if (a.order <= kNegInf) return;  // nothing but excluded tokens so far
  if (a.huge()) {
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
  int* block_max;   // [rows][steps * kStep]
  unsigned* ticket;
  int vocab, top;
  int steps;        // of a row, whatever its alignment
  long long total;  // steps of all rows
  long long run;    // steps of a CTA
};

struct ScoreShared {
  Soft soft[kScoreWarps];
  int last, n_blocks, n_cand;
  int counts[2][kScoreWarps];
  unsigned long long cand[kCand];
  int blocks[kScoreMaxTop + kScoreMaxTop / 2 + 16];
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
  // No key is above this one. (m's sign is not relied on where it is zero.)
  const unsigned long long highest = m > 0.0f && !isnan(logz) ? order_key(order(m), 0) : ~0ull;
  int turn = 0;
  if (threadIdx.x == 0) sh.n_blocks = sh.n_cand = 0;
  unsigned long long own[kOwn];
  // The blocks with the largest maxima: k of them, or more where that ends the search sooner.
#pragma unroll
  for (int i = 0; i < kOwn; i++) {
    const int b = int(threadIdx.x) + i * kScoreThreads;
    own[i] = b < r.blocks ? order_key(__ldcg(block_max + b), uint32_t(b)) : 0ull;
  }
  const int kb = min(k, r.blocks);
  // Where every thread has a block, the least of their largest has 256 >= k keys at or above it.
  unsigned long long lo = 0;
  if (r.blocks >= kScoreThreads) {
    unsigned mine = 0;
#pragma unroll
    for (int i = 0; i < kOwn; i++) mine = max(mine, unsigned(own[i] >> 32));
    mine = __reduce_min_sync(0xffffffffu, mine);
    if (lane == 0) sh.counts[1][warp] = int(mine);
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kScoreWarps; w++) mine = min(mine, unsigned(sh.counts[1][w]));
    lo = static_cast<unsigned long long>(mine) << 32;
  }
  unsigned long long bound = key_bound(kb, kb + kb / 2 + 16, lo, highest, [&](unsigned long long key) {
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
  auto collect = [&](unsigned long long least) {
    each([&](unsigned long long key) {
      if (key >= least && key) {
        const int at = atomicAdd(&sh.n_cand, 1);
        if (at < kCand) sh.cand[at] = key;
      }
    });
    __syncthreads();
  };
  // Candidates: the elements at least as large as the smallest of the picked
  // maxima (k of these exist), or all elements where there are fewer blocks than k.
  collect(r.blocks < k ? 0ull : bound & 0xFFFFFFFF00000000ull);
  if (sh.n_cand > kCand) {
    // More than there is room for (neighbours that are all large): a bound that leaves fewer.
    bound = key_bound(k, kCand, 0ull, highest, [&](unsigned long long key) {
      int c = 0;
      each([&](unsigned long long x) { c += x >= key; });
      return cta_sum(c, turn, sh);
    });
    __syncthreads();
    if (threadIdx.x == 0) sh.n_cand = 0;
    __syncthreads();
    collect(bound);
  }
  int n = sh.n_cand;
  if (n > 2 * k + 64) {
    // Ranking takes n steps a candidate: a bound among them first.
#pragma unroll
    for (int i = 0; i < kOwn; i++) {
      const int c = int(threadIdx.x) + i * kScoreThreads;
      own[i] = c < n ? sh.cand[c] : 0ull;
    }
    bound = key_bound(k, k + k / 2 + 16, 0ull, highest, [&](unsigned long long key) {
      int c = 0;
#pragma unroll
      for (int i = 0; i < kOwn; i++) c += own[i] >= key;
      return cta_sum(c, turn, sh);
    });
    __syncthreads();  // every candidate is in registers
    if (threadIdx.x == 0) sh.n_cand = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kOwn; i++)
      if (own[i] >= bound && own[i]) sh.cand[atomicAdd(&sh.n_cand, 1)] = own[i];
    __syncthreads();
    n = sh.n_cand;
  }
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
                 __shfl_xor_sync(0xffffffffu, p.t, o)};
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

__global__ void __launch_bounds__(kScoreThreads, 5) k_score(ScoreArgs a) {
  __shared__ ScoreShared sh;
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float nan = __int_as_float(0x7FC00000);
  long long g = blockIdx.x * a.run;
  const long long g1 = min(a.total, g + a.run);
  while (g < g1) {
    const size_t row = size_t(g / a.steps);
    const int s0 = int(g - (long long)row * a.steps), s1 = int(min((long long)a.steps, s0 + (g1 - g)));
    g += s1 - s0;
    const Row r(a.logits, row, a.vocab);
    int* block_max = a.top ? a.block_max + row * size_t(a.steps) * kStep : nullptr;
    // The token's logit, for whoever finishes the row: on its way while the others are read.
    float given = nan;
    if (threadIdx.x == 0) {
      const uint32_t tok = a.tokens[row];
      if (tok < uint32_t(a.vocab)) given = __ldg(r.base + r.shift + tok);
    }
    Running run;
    for (int st = s0 + warp; st < s1; st += kScoreWarps) {
      const int b = st * kStep;
      const bool whole = r.inside(b) && r.inside(b + kStep - 1);
      float4 v[kStep];
      int bm[kStep];
#pragma unroll
      for (int u = 0; u < kStep; u++) v[u] = whole ? r.load(b + u, lane) : r.load_end(b + u, lane, -INFINITY);
      add_step(run, v, bm, lane, whole, [&](int u, int j) {
        const int at = r.element(b + u, lane, j);
        return whole || (at >= 0 && at < a.vocab);
      });
      if (block_max && lane == 0) reinterpret_cast<int4*>(block_max)[st] = make_int4(bm[0], bm[1], bm[2], bm[3]);
    }
    Soft s = run.settled();
    s.s = warp_sum(s.s);
    s.t = warp_sum(s.t);
    s = soft_cta(s, warp, lane, sh);
    // Pieces of this row: those of the CTAs whose runs meet it.
    const long long c0 = (long long)row * a.steps / a.run, c1 = ((long long)(row + 1) * a.steps - 1) / a.run;
    if (c1 > c0) {
      if (threadIdx.x == 0) {
        a.part[row + blockIdx.x] = make_float4(s.m, s.s, s.t, 0.f);
        unsigned before;  // releases this CTA's writes, acquires those of the CTAs before it
        asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(before) : "l"(a.ticket + row) : "memory");
        sh.last = before == unsigned(c1 - c0);
      }
      __syncthreads();
      if (!sh.last) {
        __syncthreads();  // sh.last is read before the next piece writes it
        continue;
      }
      Soft p{-INFINITY, 0.f, 0.f};
      for (long long c = c0 + threadIdx.x; c <= c1; c += kScoreThreads) {
        const float4 q = __ldcg(a.part + row + c);
        p = soft_join(p, Soft{q.x, q.y, q.z});
      }
      s = soft_cta(soft_lanes(p, 32, lane), warp, lane, sh);
      if (threadIdx.x == 0) a.ticket[row] = 0;
    }
    const bool bad = !(s.m < INFINITY) || s.m == -INFINITY || isnan(s.s);
    const float logz = bad ? nan : log1pf(s.s);
    if (threadIdx.x == 0) {
      a.entropy[row] = logz + kLn2 * s.t / (1.0f + s.s);
      a.logprob[row] = (given - s.m) - logz;
    }
    if (a.top) alternatives(a, r, row, block_max, s.m, logz, sh);
    __syncthreads();  // shared memory is free for the next piece
  }
}

// Steps of a row, whatever its alignment.
int score_steps(size_t vocab) { return int((vocab + 3 + kStep * kBlock - 1) / (kStep * kBlock)); }

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
  const size_t blocks = size_t(tb::score_steps(vocab)) * tb::kStep;
  int per_sm = 0;
  cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, tb::k_score, tb::kScoreThreads, 0);
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
  a.steps = tb::score_steps(s->vocab);
  a.total = (long long)n * a.steps;
  // Equal runs for the CTAs that run at once.
  a.run = (a.total + s->ctas - 1) / s->ctas;
  tb::launch_pdl(tb::k_score, dim3(unsigned((a.total + a.run - 1) / a.run)), dim3(tb::kScoreThreads), 0, st, a);
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
