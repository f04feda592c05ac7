// q8_gemm.cu — the product of 8-bit rows (tb200_matmul_q8):
//
//     out[t][c] = f32(Σ_k w[c][k] · x[t][k]) · (sw[c] · sx[t])
//
// The sum is exact in 32-bit integers (|q| <= 128 and at most 131071 columns),
// so its order is free; the two f32 roundings of the scales' product and the
// final product follow it. Every variant below gives the same bits.
//
// k_matvec_q8 (few tokens): a warp per channel, dp4a on CUDA cores.
// k_gemm_q8 (more): tcgen05.mma kind::i8, s8 x s8 into s32 accumulators in
// tensor memory. Tokens are the rows of the accumulator (M = 128 a CTA),
// channels its columns (N, a multiple of 16 chosen per call). A lane then
// holds runs of one output row, and N can be fitted to the number of
// channels so that the tiles come out even over the SMs.
//   warp 0     producer: per 128 columns of K, a box of up to 128 token rows
//              and one of N channel rows (128-byte swizzle) into a ring;
//   warp 1     one lane issues the MMAs (K = 32 each), commits each stage back
//              to the producer and each tile to the epilogue;
//   warps 2-9  epilogue, two for each 32 lanes of the accumulator: tcgen05.ld, scales, then 32 x 32 outputs at a time
//              through shared memory (128-byte swizzle) into a TMA store; two
//              accumulators let it run behind the next tile's MMAs. With 32-byte
//              stores from each lane's own row it took 450 to 790 cycles for 16
//              columns, longer than the MMAs of a tile up to K = 2560.
// Persistent CTAs walk the tiles, token tiles innermost, so that a channel
// tile comes from memory once. Only the token rows that exist are loaded: the
// MMA reads whatever shared memory holds in the place of the others, and the
// accumulator rows that this makes are never read.
//
// Every mbarrier wait is bounded (kWaitCycles); on expiry the kernel leaves
// TB200_ERR_TIMEOUT in the device's async error word, lets what it issued
// drain, frees its tensor memory and returns. Every CTA takes more than half
// of an SM's shared memory, so no two share an SM and the allocation of
// tensor memory never waits.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <string>

#include "runtime.h"

namespace tb {
namespace {
constexpr size_t kMaxCols = 131071;  // 128 * 128 * 131071 < 2^31

// A warp per R channels and up to kVecTokens tokens: R rows' loads are on their
// way at once.
constexpr int kVecTokens = 4;
template <int T, int R>
__global__ void __launch_bounds__(256) k_matvec_q8(float* __restrict__ out, const int8_t* __restrict__ w,
                                                   const float* __restrict__ sw, int channels,
                                                   const int8_t* __restrict__ x, const float* __restrict__ sx, int ldw,
                                                   int ldx) {
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int c0 = (blockIdx.x * 8 + warp) * R;
  if (c0 >= channels) return;
  int acc[R][T];
  const int4* wr[R];
#pragma unroll
  for (int r = 0; r < R; r++) {
    wr[r] = reinterpret_cast<const int4*>(w + size_t(min(c0 + r, channels - 1)) * ldw);
#pragma unroll
    for (int t = 0; t < T; t++) acc[r][t] = 0;
  }
  const int n = ldw / 16;
#pragma unroll 2
  for (int i = lane; i < n; i += 32) {
    int4 a[R];
#pragma unroll
    for (int r = 0; r < R; r++) a[r] = __ldcs(wr[r] + i);
#pragma unroll
    for (int t = 0; t < T; t++) {
      const int4 b = __ldg(reinterpret_cast<const int4*>(x + size_t(t) * ldx) + i);
#pragma unroll
      for (int r = 0; r < R; r++) {
        acc[r][t] = __dp4a(a[r].x, b.x, acc[r][t]);
        acc[r][t] = __dp4a(a[r].y, b.y, acc[r][t]);
        acc[r][t] = __dp4a(a[r].z, b.z, acc[r][t]);
        acc[r][t] = __dp4a(a[r].w, b.w, acc[r][t]);
      }
    }
  }
  int mine = 0;
#pragma unroll
  for (int r = 0; r < R; r++)
#pragma unroll
    for (int t = 0; t < T; t++) {
      const int s = __reduce_add_sync(0xffffffffu, acc[r][t]);
      if (lane == t * R + r) mine = s;
    }
  const int c = c0 + lane % R, t = lane / R;
  if (t < T && c < channels)
    out[size_t(t) * channels + c] = __fmul_rn(__int2float_rn(mine), __fmul_rn(sw[c], sx[t]));
}

template <int T>
void matvec_q8(tb200_device* d, float* out, const tb200_q8* w, const tb200_q8* x) {
  const int channels = int(w->rows);
  auto go = [&](auto kernel, int r) {
    launch_pdl(kernel, dim3(unsigned((channels + 8 * r - 1) / (8 * r))), dim3(256), 0, d->stream, out, w->values,
               w->scales, channels, x->values, x->scales, int(w->ld), int(x->ld));
  };
  go(k_matvec_q8<T, T == 1 ? 1 : 2>, T == 1 ? 1 : 2);
}

// ---- tensor cores ------------------------------------------------------------

constexpr int kTileM = 128;              // token rows per CTA
constexpr int kMaxN = 256;               // channels per tile
constexpr int kKB = 128;                 // K per stage: one 128-byte swizzle row
constexpr int kQThreads = 320;
constexpr int kEpiWarps = 8, kEpiThreads = 32 * kEpiWarps;
constexpr int kQTmemCols = 512;          // two accumulators of up to 256 columns
constexpr int kQMaxStages = 24;
constexpr size_t kQMinSmem = 116 * 1024;  // more than half of an SM's 228 KB
constexpr size_t kQMaxSmem = 226 * 1024;

struct QGemmArgs {
  const float* sw;
  const float* sx;
  float* out;
  int T, M, K;       // tokens, channels, columns
  int n;             // channels per tile
  int xrows;         // token rows per tile that are loaded (a multiple of 8, at most 128)
  int stages, mtiles, ntiles;
  int tma_out;       // output rows begin on 16-byte boundaries: a TMA store can write them
  int* err;
};

// The epilogue's staging: a tile of 32 tokens by 32 channels for each warp.
constexpr int kStageTile = 32 * 128;
constexpr size_t kStaging = size_t(kEpiWarps) * kStageTile;

// Shared memory after the ring and the staging: barriers full[s], empty[s], tfull[2], tempty[2],
// mdone, then the address of the tensor memory and the epilogue's scales.
struct QTail {
  uint64_t full[kQMaxStages], empty[kQMaxStages], tfull[2], tempty[2], mdone;
  uint32_t tmem;
  int ok[kEpiWarps];
  alignas(16) float sw[2][kMaxN];
};

__host__ __device__ constexpr size_t q_stage_bytes(int n, int xrows) { return size_t(n + xrows) * kKB; }
// The last stage's MMA reads 128 token rows whatever xrows is: into the staging.
static_assert(kStaging >= size_t(kTileM) * kKB, "those reads stay inside shared memory");
__host__ __device__ constexpr size_t q_ring_bytes(int n, int xrows, int stages) {
  return stages * q_stage_bytes(n, xrows);
}

__device__ __forceinline__ void q_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void q_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Shared-memory matrix descriptor of a K-major operand in rows of 128 bytes,
// 128-byte swizzle, groups of 8 rows 1024 bytes apart: start address >> 4
// [0,14), leading byte offset >> 4 [16,30) (unused here, 1), stride byte
// offset >> 4 [32,46), version 1 [46,48), layout 2 = 128-byte swizzle [61,64).
__device__ __forceinline__ uint64_t q_desc(uint32_t saddr) {
  return uint64_t((saddr & 0x3FFFFu) >> 4) | (uint64_t(1) << 16) | (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) |
         (uint64_t(2) << 61);
}
// Instruction descriptor, kind::i8: s32 accumulator [4,6) = 2, A and B signed
// ([7,10) = 1, [10,13) = 1), both K-major, N >> 3 at [17,23), M >> 4 at [24,29).
__device__ __forceinline__ uint32_t q_idesc(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | (uint32_t(n >> 3) << 17) | (uint32_t(m >> 4) << 24);
}
template <int CG>
__device__ __forceinline__ void q_mma(uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accum) {
  if constexpr (CG == 1)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
        "l"(a), "l"(b), "r"(idesc), "r"(accum)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
        "l"(a), "l"(b), "r"(idesc), "r"(accum)
        : "memory");
}
// True for one lane of the (converged) warp, the same each time.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(p));
  return p != 0;
}
// Arrives on `bar` (with a pair: on both CTAs' barrier at that place) once
// every MMA issued so far has completed.
template <int CG>
__device__ __forceinline__ void q_commit(uint64_t* bar) {
  if constexpr (CG == 1)
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
  else
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            smem_u32(bar)),
        "h"(uint16_t(3))
        : "memory");
}
// tma_load_2d into this CTA, completing on a barrier of the pair's first CTA.
__device__ __forceinline__ void tma_load_pair(void* dst, const void* map, int x, int y, uint32_t bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%2, %3}], [%4], %5;" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar), "l"(policy)
      : "memory");
}
__device__ __forceinline__ uint32_t pair_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// The address, as the pair's CTAs see it, of a shared variable in its first CTA.
__device__ __forceinline__ uint32_t in_first(const void* p) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(smem_u32(p)));
  return r;
}
// mbar_wait for arrivals from the other CTA of the pair.
__device__ __forceinline__ bool pair_wait(uint64_t* bar, uint32_t parity, int* err) {
  const long long t0 = clock64();
  for (;;) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    if (ok) return true;
    if (clock64() - t0 > kWaitCycles) {
      set_error(err, TB200_ERR_TIMEOUT);
      return false;
    }
  }
}
__device__ __forceinline__ void pair_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// 32 consecutive 32-bit columns of this warp's 32 lanes.
__device__ __forceinline__ void q_tmem_ld32(uint32_t addr, int (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
// Waits for this warp's loads from tensor memory; `r` is not read before.
__device__ __forceinline__ void q_tmem_wait(int (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 32; i++) asm volatile("" : "+r"(r[i]));
}
// Stores a box from shared memory at (x, y); its elements outside the map are left out.
__device__ __forceinline__ void tma_store_2d(const void* map, int x, int y, const void* src) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(x), "r"(y), "r"(smem_u32(src))
               : "memory");
}

// CG CTAs work on a tile of 128 CG tokens by n channels. A pair (CG = 2) sits
// on neighbouring SMs: each CTA loads its 128 tokens and half of the channels,
// the first one's MMA warp issues MMAs of 256 tokens over both CTAs' shared
// memory, and each CTA finds its tokens' sums in its own tensor memory. Per
// output that takes two thirds of one CTA's bytes from L2, which is what
// bounds many tokens.
template <int CG>
__global__ void __launch_bounds__(kQThreads, 1)
    k_gemm_q8(const __grid_constant__ CUtensorMap tw, const __grid_constant__ CUtensorMap tx,
              const __grid_constant__ CUtensorMap tout, const __grid_constant__ CUtensorMap tout16, QGemmArgs a) {
  extern __shared__ unsigned char smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  unsigned char* sm = smem_raw + (((raw + 1023u) & ~1023u) - raw);  // swizzled tiles: 1024-byte alignment
  const int stages = a.stages, n = a.n, wrows = n / CG;
  const uint32_t stage_bytes = uint32_t(q_stage_bytes(wrows, a.xrows));
  unsigned char* staging = sm + q_ring_bytes(wrows, a.xrows, stages);
  QTail& tl = *reinterpret_cast<QTail*>(staging + kStaging);
  const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int rank = CG == 2 ? int(pair_rank()) : 0;
  const int group = int(blockIdx.x) / CG, groups = int(gridDim.x) / CG;
  const int nkb = (a.K + kKB - 1) / kKB;
  const int tiles = a.mtiles * a.ntiles;
  // Each group begins its sums at another place of K: the order is free, and
  // CTAs that share token rows do not all ask the same L2 slices for them at once.
  const int k0 = int((long long)group * nkb / groups);

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; s++) {
      mbar_init(&tl.full[s], 1);
      mbar_init(&tl.empty[s], 1);
    }
    for (int b = 0; b < 2; b++) {
      mbar_init(&tl.tfull[b], 1);
      mbar_init(&tl.tempty[b], kEpiWarps * CG);  // one arrival per epilogue warp
    }
    mbar_init(&tl.mdone, 1);
    fence_mbar_init();
  }
  if (warp == 1) {
    if constexpr (CG == 1) {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tl.tmem)),
                   "r"(kQTmemCols)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tl.tmem)),
                   "r"(kQTmemCols)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
  }
  if (threadIdx.x == 32 * 2) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tw)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tx)) : "memory");
  }
  q_fence_before();
  __syncthreads();
  if constexpr (CG == 2) pair_sync();  // both CTAs' barriers and tensor memory are there
  q_fence_after();
  const uint32_t tmem = tl.tmem;
  pdl_launch_dependents();
  pdl_wait();

  // The producer's and the MMA warp's lanes stay together and one of them is
  // elected at each instruction: what they issue takes uniform registers, and
  // in a branch of one lane the compiler has to move every operand there
  // (64 x 19456 x 2560: 10.9 us instead of 7.3).
  if (warp == 0) {
    const uint64_t pol_w = l2_evict_first(), pol_x = l2_evict_last();
    int i = 0, s = 0;
    uint32_t phase = 1;
    bool ok = true;
    for (int tile = group; tile < tiles && ok; tile += groups) {
      const int m0 = (tile % a.mtiles * CG + rank) * kTileM, n0 = tile / a.mtiles * n + rank * wrows;
      for (int k = 0; k < nkb; k++, i++) {
        if (!mbar_wait(&tl.empty[s], phase, a.err)) {
          ok = false;
          break;
        }
        const int at = (k + k0 < nkb ? k + k0 : k + k0 - nkb) * kKB;
        unsigned char *dw = sm + size_t(s) * stage_bytes, *dx = dw + size_t(wrows) * kKB;
        if (elect_one()) {
          // The first CTA's barrier counts both CTAs' bytes, of which the second's may come before it
          // expects them.
          if (rank == 0) mbar_arrive_expect_tx(&tl.full[s], CG * stage_bytes);
          if constexpr (CG == 1) {
            tma_load_2d(dw, &tw, at, n0, &tl.full[s], pol_w);
            tma_load_2d(dx, &tx, at, m0, &tl.full[s], pol_x);
          } else {
            const uint32_t bar = in_first(&tl.full[s]);
            tma_load_pair(dw, &tw, at, n0, bar, pol_w);
            tma_load_pair(dx, &tx, at, m0, bar, pol_x);
          }
        }
        if (++s == stages) s = 0, phase ^= 1;
      }
    }
    // Every issued copy has landed before the CTA can exit: it has been waited
    // for, or (the second CTA's) read.
    for (int j = i - 1; j >= 0 && j >= i - stages; j--)
      mbar_wait(rank == 0 ? &tl.full[j % stages] : &tl.empty[j % stages], (j / stages) & 1, nullptr);
  } else if (warp == 1) {
    if (rank == 0) {
      const uint32_t idesc = q_idesc(CG * kTileM, n);
      const uint64_t desc0 = q_desc(smem_u32(sm));
      int s = 0, ti = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = group; tile < tiles && ok; tile += groups, ti++) {
        const int b = ti & 1;
        // The epilogue has drained this accumulator's previous tile.
        const uint32_t drained = ((ti >> 1) - 1) & 1;
        if (!(CG == 1 ? mbar_wait(&tl.tempty[b], drained, a.err) : pair_wait(&tl.tempty[b], drained, a.err))) break;
        q_fence_after();
        const uint32_t acc = tmem + uint32_t(b * kMaxN);
        for (int k = 0; k < nkb; k++) {
          if (!mbar_wait(&tl.full[s], phase, a.err)) {
            ok = false;
            break;
          }
          q_fence_after();
          const uint64_t db = desc0 + ((s * stage_bytes) >> 4), da = db + ((uint32_t(wrows) * kKB) >> 4);
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < kKB / 32; kk++)
              q_mma<CG>(acc, da + 2 * kk, db + 2 * kk, idesc, (k > 0 || kk > 0) ? 1u : 0u);
            q_commit<CG>(&tl.empty[s]);
          }
          if (++s == stages) s = 0, phase ^= 1;
        }
        if (ok && elect_one()) q_commit<CG>(&tl.tfull[b]);
      }
      // Tensor memory is freed below only after every MMA has completed.
      if (elect_one()) q_commit<CG>(&tl.mdone);
      mbar_wait(&tl.mdone, 0, nullptr);
    }
  } else {
    const int q = warp & 3;  // the 32 accumulator lanes this warp can read
    const int e = int(threadIdx.x) - 64;
    int ti = 0;
    // This lane's row of the warp's staging tile: 16-byte piece j lies at j ^ (row & 7).
    unsigned char* tile_s = staging + (warp - 2) * kStageTile;
    float4* mine_s = reinterpret_cast<float4*>(tile_s + lane * 128);
    // The scales of a tile are fetched while the one before is written.
    static_assert(kEpiThreads == kMaxN, "a channel's scale for each thread");
    float next_sw = 0.f, next_sx = 0.f;
    auto fetch = [&](int tile) {
      if (tile >= tiles) return;
      const int t = (tile % a.mtiles * CG + rank) * kTileM + 32 * q + lane, c = tile / a.mtiles * n + e;
      next_sw = e < n && c < a.M ? a.sw[c] : 0.f;
      next_sx = t < a.T ? a.sx[t] : 0.f;
    };
    fetch(group);
    for (int tile = group; tile < tiles; tile += groups, ti++) {
      const int b = ti & 1;
      const int m0 = (tile % a.mtiles * CG + rank) * kTileM, n0 = tile / a.mtiles * n;
      const int cols = min(n, a.M - n0);
      tl.sw[b][e] = next_sw;
      const float sx = next_sx;
      fetch(tile + groups);
      // The warps take the same way out: a verdict is shared. The barriers
      // also put tl.sw in place.
      const bool mine = __all_sync(0xffffffffu, mbar_wait(&tl.tfull[b], (ti >> 1) & 1, a.err));
      if (lane == 0) tl.ok[warp - 2] = mine;
      named_sync(1, kEpiThreads);
      const bool ok = __all_sync(0xffffffffu, tl.ok[lane % kEpiWarps] != 0);
      named_sync(1, kEpiThreads);
      if (!ok) break;
      q_fence_after();
      const uint32_t taddr = tmem + uint32_t(b * kMaxN) + (uint32_t(32 * q) << 16);
      // 32 tokens by (up to) 32 channels from column c.
      auto put = [&](int c, int (&acc)[32]) {
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");  // the tile's last store
        __syncwarp();
        const bool half = c + 32 > n;  // the tile ends after 16 channels: rows of 64 bytes, not swizzled
        float4* to_s = half ? reinterpret_cast<float4*>(tile_s + lane * 64) : mine_s;
        const int flip = half ? 0 : lane & 7;
#pragma unroll
        for (int j = 0; j < 8; j++) {
          if (half && j >= 4) break;
          const float4 sw = *reinterpret_cast<const float4*>(&tl.sw[b][c + 4 * j]);
          to_s[j ^ flip] = make_float4(__fmul_rn(__int2float_rn(acc[4 * j]), __fmul_rn(sw.x, sx)),
                                       __fmul_rn(__int2float_rn(acc[4 * j + 1]), __fmul_rn(sw.y, sx)),
                                       __fmul_rn(__int2float_rn(acc[4 * j + 2]), __fmul_rn(sw.z, sx)),
                                       __fmul_rn(__int2float_rn(acc[4 * j + 3]), __fmul_rn(sw.w, sx)));
        }
        if (a.tma_out) fence_proxy_async_smem();
        __syncwarp();
        if (a.tma_out) {
          if (lane == 0) {
            tma_store_2d(half ? &tout16 : &tout, n0 + c, m0 + 32 * q, tile_s);
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          }
        } else if (c + lane < cols) {
          const int rows = min(32, a.T - m0 - 32 * q), pitch = half ? 64 : 128;
          float* to = a.out + size_t(m0 + 32 * q) * a.M + n0 + c + lane;
          for (int r = 0; r < rows; r++, to += a.M)
            *to = *reinterpret_cast<const float*>(tile_s + r * pitch + (((lane >> 2) ^ (half ? 0 : r & 7)) << 4) +
                                                  (lane & 3) * 4);
        }
        __syncwarp();
      };
      if (m0 + 32 * q < a.T) {  // warp-uniform: some of this warp's tokens exist
        // Every second 32 channels are this warp's; the next ones are on their way while it writes these.
        constexpr int kNext = 32 * (kEpiWarps / 4);
        int acc[2][32];
        int c = 32 * ((warp - 2) / 4);
        if (c < cols) q_tmem_ld32(taddr + c, acc[0]);
        while (c < cols) {
          q_tmem_wait(acc[0]);
          if (c + kNext < cols) q_tmem_ld32(taddr + c + kNext, acc[1]);
          put(c, acc[0]);
          if ((c += kNext) >= cols) break;
          q_tmem_wait(acc[1]);
          if (c + kNext < cols) q_tmem_ld32(taddr + c + kNext, acc[0]);
          put(c, acc[1]);
          c += kNext;
        }
      }
      q_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (CG == 1)
          mbar_arrive(&tl.tempty[b]);
        else
          asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(in_first(&tl.tempty[b]))
                       : "memory");
      }
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");  // shared memory may go
  }
  q_fence_before();
  __syncthreads();
  if constexpr (CG == 2) pair_sync();  // no MMA reads the other CTA's memory, no arrival is on its way there
  if (warp == 1) {
    q_fence_after();
    if constexpr (CG == 1)
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kQTmemCols) : "memory");
    else
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kQTmemCols) : "memory");
  }
}

// Tensor map of `rows` rows of `cols` elements, `pitch` bytes apart.
int encode_tmap(CUtensorMap* map, CUtensorMapDataType type, void* base, size_t rows, size_t cols, size_t pitch,
                int box_cols, int box_rows, CUtensorMapSwizzle swizzle = CU_TENSOR_MAP_SWIZZLE_128B) {
  static PFN_cuTensorMapEncodeTiled_v12000 encode = [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult r{};
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &r) != cudaSuccess ||
        r != cudaDriverEntryPointSuccess)
      fn = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
  }();
  if (!encode) return rt::fail(TB200_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
  cuuint64_t dims[2] = {cuuint64_t(cols), cuuint64_t(rows)};
  cuuint64_t strides[1] = {cuuint64_t(pitch)};
  cuuint32_t box[2] = {cuuint32_t(box_cols), cuuint32_t(box_rows)};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = encode(map, type, 2, base, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                      swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return rt::fail(TB200_ERR_CUDA, "matmul_q8: cuTensorMapEncodeTiled failed (" + std::to_string(int(r)) + ")");
  return TB200_OK;
}
int encode_tmap_q8(CUtensorMap* map, const tb200_q8* q, int box_rows) {
  return encode_tmap(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, q->values, q->cap, q->ld, q->ld, kKB, box_rows);
}

// Channels per tile: the multiple of `step` with which the group that has most
// to do has least, a tile's fixed cost (filling the ring, the last tile's
// epilogue) counted as 24 channels.
int plan_n(int M, int mtiles, int groups, int step) {
  int best = 0;
  long long least = 0;
  for (int n = step; n <= kMaxN; n += step) {
    const long long tiles = (long long)mtiles * ((M + n - 1) / n);
    const long long cost = (tiles + groups - 1) / groups * (n + 24);
    if (!best || cost <= least) best = n, least = cost;
  }
  return best;
}

template <int CG>
int gemm_q8(tb200_device* d, float* out, const tb200_q8* w, const tb200_q8* x) {
  QGemmArgs a{};
  a.sw = w->scales;
  a.sx = x->scales;
  a.out = out;
  a.T = int(x->rows);
  a.M = int(w->rows);
  a.K = int(w->cols);
  a.err = d->async_err_dev;
  a.mtiles = (a.T + CG * kTileM - 1) / (CG * kTileM);
  a.n = plan_n(a.M, a.mtiles, d->sms / CG, 16 * CG);
  if (getenv("TBN")) a.n = atoi(getenv("TBN"));
  a.ntiles = (a.M + a.n - 1) / a.n;
  a.xrows = CG == 2 ? kTileM : std::min(kTileM, (a.T + 7) / 8 * 8);
  const int wrows = a.n / CG;
  const size_t fixed = kStaging + sizeof(QTail) + 1024;
  a.stages = int(std::min<size_t>(kQMaxStages, (kQMaxSmem - fixed) / q_stage_bytes(wrows, a.xrows)));
  a.tma_out = reinterpret_cast<uintptr_t>(out) % 16 == 0 && a.M % 4 == 0;
  CUtensorMap tw, tx, tout{}, tout16{};
  if (int rc = encode_tmap_q8(&tw, w, wrows)) return rc;
  if (int rc = encode_tmap_q8(&tx, x, a.xrows)) return rc;
  if (a.tma_out) {
    const auto f32 = CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
    if (int rc = encode_tmap(&tout, f32, out, x->rows, w->rows, w->rows * 4, 32, 32)) return rc;
    if (a.n % 32)
      if (int rc = encode_tmap(&tout16, f32, out, x->rows, w->rows, w->rows * 4, 16, 32, CU_TENSOR_MAP_SWIZZLE_NONE))
        return rc;
  }
  const size_t smem = std::max(kQMinSmem, q_ring_bytes(wrows, a.xrows, a.stages) + fixed);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(CG * std::min<long long>((long long)a.mtiles * a.ntiles, d->sms / CG)));
  cfg.blockDim = dim3(kQThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = d->stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim = {CG, 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = CG;  // one CTA: no cluster
  cudaLaunchKernelEx(&cfg, k_gemm_q8<CG>, tw, tx, tout, tout16, a);
  return rt::launched("matmul_q8");
}

}  // namespace

cudaError_t init_q8_kernels() {
  cudaError_t e = cudaFuncSetAttribute(k_gemm_q8<1>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(kQMaxSmem));
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(k_gemm_q8<2>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(kQMaxSmem));
  return e;
}

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
  switch (x->rows) {
    case 1: tb::matvec_q8<1>(d, out->ptr, w, x); break;
    case 2: tb::matvec_q8<2>(d, out->ptr, w, x); break;
    case 3: tb::matvec_q8<3>(d, out->ptr, w, x); break;
    case 4: tb::matvec_q8<4>(d, out->ptr, w, x); break;
    default: return x->rows > 128 && !getenv("TB1") ? tb::gemm_q8<2>(d, out->ptr, w, x) : tb::gemm_q8<1>(d, out->ptr, w, x);
  }
  return rt::launched("matmul_q8");
}

}  // extern "C"
