// q8_gemm.cu — the product of 8-bit rows (tb200_matmul_q8):
//
//     out[t][c] = f32(Σ_k w[c][k] · x[t][k]) · (sw[c] · sx[t])
//
// The sum is exact in 32-bit integers (|q| <= 128 and at most 131071 columns),
// so its order is free; the two f32 roundings of the scales' product and the
// final product follow it. Every variant below gives the same bits.
//
// k_matvec_q8 (up to eight tokens over few weights): a warp per channel, dp4a on CUDA cores.
// k_gemm_q8 (more): tcgen05.mma kind::i8, s8 x s8 into s32 accumulators in
// tensor memory. Tokens are the rows of the accumulator (M = 128 a CTA),
// channels its columns (N, a multiple of 16 chosen per call). A lane then
// holds runs of one output row, and N can be fitted to the number of
// channels so that the tiles come out even over the SMs.
//   warp 0     producer: per 128 columns of K, a box of up to 128 token rows
//              and one of N channel rows (128-byte swizzle) into a ring;
//   warp 1     issues the MMAs (K = 32 each), commits each stage back to the
//              producer and each tile to the epilogue;
//   warps 2-9  epilogue, two for each 32 lanes of the accumulator: tcgen05.ld,
//              scales, then 32 x 32 outputs at a time through shared memory
//              (128-byte swizzle) into a TMA store; two accumulators let it run
//              behind the next tile's MMAs. With 32-byte stores from each lane's
//              own row it took 450 to 790 cycles for 16 columns, longer than
//              the MMAs of a tile up to K = 2560.
// Persistent CTAs walk the tiles, token tiles innermost, so that a channel
// tile comes from memory once; many tokens go to pairs of CTAs, long sums over
// few channels to clusters that share a tile's K (below). Only the token rows
// that exist are loaded: the MMA reads whatever shared memory holds in the place
// of the others, and the accumulator rows that this makes are never read.
//
// Measured (us; memory or bf16-rate floor): 64 x 19456 x 2560 11.6 (8.5), of which
// filling the ring and the last tile's way out take 3; 1999 x 9728 x 2560 43.8 (58.8;
// 2.3 P operations/s, bound by the 50 to 70 bytes a clock that a SM's loads reach),
// 51 back to back under the power cap; 64 x 2560 x 9728 9.5 (4.1).
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

// S warps per R channels, for T tokens. Rows are read in the order they lie in
// memory by many warps with two 16-byte pieces each on their way: six or eight
// of them, or more channels a warp, are slower (one token, 151936 x 1024: 24.3 us,
// 27.4 with predicated batches; 2560 x 9728: 7.8 and 9.7).
template <int T, int R, int S>
__global__ void __launch_bounds__(256) k_matvec_q8(float* out, const int8_t* w, const float* sw, int channels,
                                                   const int8_t* x, const float* sx, int ldw, int ldx) {
  pdl_launch_dependents();
  pdl_wait();
  w = after_wait(w), x = after_wait(x);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int c0 = (blockIdx.x * 8 + warp) / S * R;
  if (S == 1 && c0 >= channels) return;
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
  for (int i = lane + 32 * (warp % S); i < n; i += 32 * S) {
    int4 a[R];
#pragma unroll
    for (int r = 0; r < R; r++) a[r] = ld_stream_s32x4(wr[r] + i);
    // Every token's piece before the first product (8 x 1024 x 1024: 2.6 us with loads and products in turns, 1.9).
    int4 b[T];
#pragma unroll
    for (int t = 0; t < T; t++) b[t] = ld_s32x4(reinterpret_cast<const int4*>(x + size_t(t) * ldx) + i);
#pragma unroll
    for (int t = 0; t < T; t++)
#pragma unroll
      for (int r = 0; r < R; r++) {
        acc[r][t] = __dp4a(a[r].x, b[t].x, acc[r][t]);
        acc[r][t] = __dp4a(a[r].y, b[t].y, acc[r][t]);
        acc[r][t] = __dp4a(a[r].z, b[t].z, acc[r][t]);
        acc[r][t] = __dp4a(a[r].w, b[t].w, acc[r][t]);
      }
  }
  int mine = 0;  // lane t R + r: channel r, token t
#pragma unroll
  for (int r = 0; r < R; r++)
#pragma unroll
    for (int t = 0; t < T; t++) {
      const int s = __reduce_add_sync(0xffffffffu, acc[r][t]);
      if (lane == t * R + r) mine = s;
    }
  if constexpr (S > 1) {
    __shared__ int parts[8][R * T];
    if (lane < R * T) parts[warp][lane] = mine;
    __syncthreads();
    if (warp % S) return;
    if (lane < R * T)
      for (int s = 1; s < S; s++) mine += parts[warp + s][lane];
  }
  const int c = c0 + lane % R, t = lane / R;
  if (t < T && c < channels)
    out[size_t(t) * channels + c] = __fmul_rn(__int2float_rn(mine), __fmul_rn(sw[c], sx[t]));
}

template <int T>
void matvec_q8(tb200_device* d, float* out, const tb200_q8* w, const tb200_q8* x) {
  const int channels = int(w->rows);
  // One channel a warp for one token, two for more, which halves the reads of x.
  constexpr int R = T == 1 ? 1 : 2;
  auto go = [&](auto kernel, int s) {
    const int each = 8 / s * R;  // channels of a block
    launch_pdl(kernel, dim3(unsigned((channels + each - 1) / each)), dim3(256), 0, d->stream, out, w->values, w->scales,
               channels, x->values, x->scales, int(w->ld), int(x->ld));
  };
  // Two, four or eight warps share the rows where there would be fewer than 28, 8 or 4 warps an SM (us: one
  // token, 2560 x 9728 7.7 with one and 5.9 with two, 6000 x 4096 5.6 and 5.9; four tokens, 2560 x 2560 3.6 with
  // two and 4.4 with four; 1000 x 20000 with two, four and eight, one token 7.9, 5.7 and 4.7, four tokens 14.8,
  // 8.5 and 5.8; 1024 x 1024, one token, 1.4, 1.4 and 1.8).
  if (channels / R < 4 * d->sms)
    go(k_matvec_q8<T, R, 8>, 8);
  else if (channels / R < 8 * d->sms)
    go(k_matvec_q8<T, R, 4>, 4);
  else if (channels / R < 28 * d->sms)
    go(k_matvec_q8<T, R, 2>, 2);
  else
    go(k_matvec_q8<T, R, 1>, 1);
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
  int splits;        // SPLIT: CTAs that share a tile's sums
  int tma_out;       // output rows begin on 16-byte boundaries: a TMA store can write them
  unsigned ring;     // bytes of the ring
  unsigned recv;     // SPLIT: bytes of the other CTAs' sums
  int* err;
};

// The epilogue's staging: a tile of 32 tokens by 32 channels for each warp.
constexpr int kStageTile = 32 * 128;
constexpr size_t kStaging = size_t(kEpiWarps) * kStageTile;

// Shared memory after the ring, the staging and what a split tile receives:
// barriers, then the address of the tensor memory and the epilogue's scales.
struct QTail {
  uint64_t full[kQMaxStages], empty[kQMaxStages], tfull[2], tempty[2], mdone, summed;
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
// The same verdict for the whole warp.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int* err) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, err));
}
__device__ __forceinline__ void cluster_sync() {
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

// Copies from this CTA's shared memory to the same cluster's CTA `rank`,
// completing on a barrier there.
__device__ __forceinline__ void bulk_to_cta(const void* dst, const void* src, uint32_t bytes, const uint64_t* bar,
                                            uint32_t rank) {
  uint32_t d, b;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(d) : "r"(smem_u32(dst)), "r"(rank));
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(b) : "r"(smem_u32(bar)), "r"(rank));
  asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(d),
               "r"(smem_u32(src)), "r"(bytes), "r"(b)
               : "memory");
}

// CG CTAs work on a tile of 128 CG tokens by n channels. A pair (CG = 2) sits
// on neighbouring SMs: each CTA loads its 128 tokens and half of the channels,
// the first one's MMA warp issues MMAs of 256 tokens over both CTAs' shared
// memory, and each CTA finds its tokens' sums in its own tensor memory. Per
// output that takes two thirds of one CTA's bytes from L2, which is what
// bounds many tokens.
//
// SPLIT: the sums of a tile are cut over the CTAs of a cluster (a.splits of
// them), one tile a cluster. An MMA takes at least 64 cycles, the time to read
// its 128 token rows, so narrow tiles over all of a long K waste it. The CTAs
// take turns in the tile's units of 32 tokens by 32 channels: each copies its
// sums of a unit to the unit's CTA (4 KB by a bulk copy; reading them there
// word by word took 13000 cycles), which adds them up and writes them.
template <int CG, bool SPLIT>
__global__ void __launch_bounds__(kQThreads, 1)
    k_gemm_q8(const __grid_constant__ CUtensorMap tw, const __grid_constant__ CUtensorMap tx,
              const __grid_constant__ CUtensorMap tout, const __grid_constant__ CUtensorMap tout16, QGemmArgs a) {
  extern __shared__ unsigned char smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  unsigned char* sm = smem_raw + (((raw + 1023u) & ~1023u) - raw);  // swizzled tiles: 1024-byte alignment
  const int stages = a.stages, n = a.n, wrows = n / CG;
  const uint32_t stage_bytes = uint32_t(q_stage_bytes(wrows, a.xrows));
  unsigned char* staging = sm + a.ring;
  unsigned char* recv = staging + kStaging;  // SPLIT: the other CTAs' sums, [this CTA's units][CTA]
  QTail& tl = *reinterpret_cast<QTail*>(recv + a.recv);
  const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  static_assert(CG == 1 || !SPLIT, "a split tile is one CTA wide");
  const int rank = CG == 2 ? int(pair_rank()) : 0;
  const int per = SPLIT ? a.splits : CG, part = SPLIT ? int(pair_rank()) : 0;
  const int group = int(blockIdx.x) / per, groups = int(gridDim.x) / per;
  // The 128-column steps of K of this CTA: kb0 .. kb0 + nkb.
  const int all_kb = (a.K + kKB - 1) / kKB;
  const int kb0 = SPLIT ? int((long long)all_kb * part / a.splits) : 0;
  const int nkb = SPLIT ? int((long long)all_kb * (part + 1) / a.splits) - kb0 : all_kb;
  const int tiles = a.mtiles * a.ntiles;
  // SPLIT: units of the tile, quarter by quarter of its tokens within 32 channels.
  const int quarters = SPLIT ? (min(kTileM, a.T - group % a.mtiles * kTileM) + 31) / 32 : 0;
  const int units = SPLIT ? (min(n, a.M - group / a.mtiles * n) + 31) / 32 * quarters : 0;
  // Each group begins its sums at another place of K: the order is free, and
  // CTAs that share token rows do not all ask the same L2 slices for them at once.
  const int k0 = SPLIT ? 0 : int((long long)group * nkb / groups);

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
    if constexpr (SPLIT) {
      mbar_init(&tl.summed, 1);
      const int mine = (units - part + a.splits - 1) / a.splits;
      mbar_arrive_expect_tx(&tl.summed, uint32_t(mine * (a.splits - 1) * kStageTile));
    }
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
  if constexpr (CG == 2 || SPLIT) cluster_sync();  // every CTA's barriers and tensor memory are there
  q_fence_after();
  const uint32_t tmem = tl.tmem;
  pdl_launch_dependents();
  pdl_wait();

  // Epilogue warps: scales and writes the sums of 32 tokens (quarter q of the
  // tile at m0) by up to 32 channels from column c of the tile at n0, a lane a
  // token, through this warp's staging tile, where 16-byte piece j of a row
  // lies at j ^ (row & 7). b: which of tl.sw.
  unsigned char* tile_s = staging + (warp - 2) * kStageTile;
  float4* mine_s = reinterpret_cast<float4*>(tile_s + lane * 128);
  auto put = [&](int b, int m0, int n0, int q, int c, float sx, int (&acc)[32]) {
    const int cols = min(n, a.M - n0);
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
        if (!warp_wait(&tl.empty[s], phase, a.err)) {
          ok = false;
          break;
        }
        const int at = (kb0 + (k + k0 < nkb ? k + k0 : k + k0 - nkb)) * kKB;
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
        if (!(CG == 1 ? warp_wait(&tl.tempty[b], drained, a.err)
                      : __all_sync(0xffffffffu, pair_wait(&tl.tempty[b], drained, a.err))))
          break;
        q_fence_after();
        const uint32_t acc = tmem + uint32_t(b * kMaxN);
        for (int k = 0; k < nkb; k++) {
          if (!warp_wait(&tl.full[s], phase, a.err)) {
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
      const bool mine = warp_wait(&tl.tfull[b], (ti >> 1) & 1, a.err);
      if (lane == 0) tl.ok[warp - 2] = mine;
      named_sync(1, kEpiThreads);
      const bool ok = __all_sync(0xffffffffu, tl.ok[lane % kEpiWarps] != 0);
      named_sync(1, kEpiThreads);
      if (!ok) break;
      q_fence_after();
      const uint32_t taddr = tmem + uint32_t(b * kMaxN) + (uint32_t(32 * q) << 16);
      if (m0 + 32 * q < a.T) {  // warp-uniform: some of this warp's tokens exist
        // Every second 32 channels are this warp's; the next ones are on their way while it writes these.
        constexpr int kNext = 32 * (kEpiWarps / 4);
        int acc[2][32];
        int c = 32 * ((warp - 2) / 4);
        auto give = [&](int (&v)[32]) {
          if constexpr (SPLIT) {
            // Where the ring was: every load has landed and every MMA has read it.
            const int u = c / 32 * quarters + q, owner = u % a.splits;
            unsigned char* sums = sm + size_t(u) * kStageTile;
            int4* to = reinterpret_cast<int4*>(sums + lane * 128);
#pragma unroll
            for (int j = 0; j < 8; j++)
              to[j ^ (lane & 7)] = make_int4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
            fence_proxy_async_smem();
            __syncwarp();
            if (owner != part && lane == 0)
              bulk_to_cta(recv + size_t(u / a.splits * a.splits + part) * kStageTile, sums, kStageTile, &tl.summed,
                          uint32_t(owner));
          } else {
            put(b, m0, n0, q, c, sx, v);
          }
        };
        if (c < cols) q_tmem_ld32(taddr + c, acc[0]);
        while (c < cols) {
          q_tmem_wait(acc[0]);
          if (c + kNext < cols) q_tmem_ld32(taddr + c + kNext, acc[1]);
          give(acc[0]);
          if ((c += kNext) >= cols) break;
          q_tmem_wait(acc[1]);
          if (c + kNext < cols) q_tmem_ld32(taddr + c + kNext, acc[0]);
          give(acc[1]);
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
  }
  if constexpr (SPLIT) {
    __syncthreads();  // this CTA's own sums are in its shared memory
    if (warp >= 2 && warp_wait(&tl.summed, 0, a.err)) {
      const int m0 = group % a.mtiles * kTileM, n0 = group / a.mtiles * n;
      for (int i = warp - 2; part + i * a.splits < units; i += kEpiWarps) {
        const int u = part + i * a.splits, q = u % quarters, c = u / quarters * 32, t = m0 + 32 * q + lane;
        int acc[32];
#pragma unroll
        for (int j = 0; j < 32; j++) acc[j] = 0;
        for (int r = 0; r < a.splits; r++) {
          const unsigned char* from =
              r == part ? sm + size_t(u) * kStageTile : recv + size_t(i * a.splits + r) * kStageTile;
#pragma unroll
          for (int j = 0; j < 8; j++) {
            const int4 v = *reinterpret_cast<const int4*>(from + lane * 128 + ((j ^ (lane & 7)) << 4));
            acc[4 * j] += v.x, acc[4 * j + 1] += v.y, acc[4 * j + 2] += v.z, acc[4 * j + 3] += v.w;
          }
        }
        put(0, m0, n0, q, c, t < a.T ? a.sx[t] : 0.f, acc);
      }
    }
  }
  if (warp >= 2 && lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");  // shared memory may go
  q_fence_before();
  __syncthreads();
  // The first CTA's last commit arrives here too, which nothing above has waited for: not in shared memory that
  // may be another kernel's by then.
  if (CG == 2 && rank == 1 && warp == 1) mbar_wait(&tl.mdone, 0, nullptr);
  if constexpr (CG == 2 || SPLIT) cluster_sync();  // nothing reads or signals the other CTAs' memory any more
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

struct QPlan {
  int n, splits;
};
// One CTA a tile: the channels (a multiple of 16) with which the CTA that has
// most to do has least, a tile's fixed cost (filling the ring, the last tile's
// epilogue) counted as 24 channels. Where the tiles leave SMs idle, the sums
// may be cut over two or four CTAs instead: in cycles, a step of K takes four MMAs
// of n / 2, at least 64, and a cluster and its adding up about 5000 (64 x 2560 x
// 9728: 14.2 us uncut, 9.5 cut over four; 64 x 1024 x 2048: 4.9 and 5.7). Clusters
// of eight CTAs of this size do not all run at once: 18 and 10.7 us.
constexpr size_t kQFixed = kStaging + sizeof(QTail) + 1024;
// Bytes of sums that a CTA of a split tile receives, by the quarters of its tokens.
size_t q_recv_bytes(int n, int splits, int quarters) {
  const int units = (n + 31) / 32 * quarters;
  return size_t((units + splits - 1) / splits) * splits * kStageTile;
}
int q_stages(int wrows, int xrows, size_t recv) {
  return int(std::min<size_t>(kQMaxStages, (kQMaxSmem - kQFixed - recv) / q_stage_bytes(wrows, xrows)));
}
QPlan plan_one(int M, int nkb, int T, int sms) {
  const int mtiles = (T + kTileM - 1) / kTileM, xrows = std::min(kTileM, (T + 7) / 8 * 8), quarters = (xrows + 31) / 32;
  QPlan best{0, 1};
  long long least = 0;
  for (int n = 16; n <= kMaxN; n += 16) {
    const long long tiles = (long long)mtiles * ((M + n - 1) / n);
    const long long cost = (tiles + sms - 1) / sms * (n + 24);
    if (!best.n || cost <= least) best.n = n, least = cost;
  }
  const long long tiles = (long long)mtiles * ((M + best.n - 1) / best.n);
  long long cycles = (tiles + sms - 1) / sms * nkb * 4 * std::max(64, best.n / 2);
  for (int splits = 2; splits <= 4 && splits <= nkb; splits *= 2)
    for (int n = 32; n <= 160; n += 16) {
      if (q_stages(n, xrows, q_recv_bytes(n, splits, quarters)) < 3) continue;
      // A cluster lies within one of the groups of SMs that a GPU is made of, which it need not divide.
      if ((long long)mtiles * ((M + n - 1) / n) * splits > sms - sms * splits / 64) continue;
      const long long c = (long long)((nkb + splits - 1) / splits) * 4 * std::max(64, n / 2) + 5000;
      if (c < cycles) best = {n, splits}, cycles = c;
    }
  return best;
}
// Pairs of CTAs (n a multiple of 32): bound by loads, so a step counts as its rows.
QPlan plan_pair(int M, int mtiles, int pairs) {
  QPlan best{0, 1};
  long long least = 0;
  for (int n = 32; n <= kMaxN; n += 32) {
    const long long tiles = (long long)mtiles * ((M + n - 1) / n);
    const long long cost = (tiles + pairs - 1) / pairs * (n / 2 + kTileM);
    if (!best.n || cost <= least) best.n = n, least = cost;
  }
  return best;
}

template <int CG, bool SPLIT>
int launch_gemm_q8(tb200_device* d, QGemmArgs a, QPlan p, const tb200_q8* w, const tb200_q8* x) {
  a.mtiles = (a.T + CG * kTileM - 1) / (CG * kTileM);
  a.n = p.n;
  a.splits = p.splits;
  a.ntiles = (a.M + a.n - 1) / a.n;
  a.xrows = CG == 2 ? kTileM : std::min(kTileM, (a.T + 7) / 8 * 8);
  const int wrows = a.n / CG;
  a.recv = SPLIT ? unsigned(q_recv_bytes(a.n, a.splits, (a.xrows + 31) / 32)) : 0;
  a.stages = q_stages(wrows, a.xrows, a.recv);
  CUtensorMap tw, tx, tout{}, tout16{};
  if (int rc = encode_tmap_q8(&tw, w, wrows)) return rc;
  if (int rc = encode_tmap_q8(&tx, x, a.xrows)) return rc;
  if (a.tma_out) {
    const auto f32 = CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
    if (int rc = encode_tmap(&tout, f32, a.out, x->rows, w->rows, w->rows * 4, 32, 32)) return rc;
    if (a.n % 32)
      if (int rc = encode_tmap(&tout16, f32, a.out, x->rows, w->rows, w->rows * 4, 16, 32, CU_TENSOR_MAP_SWIZZLE_NONE))
        return rc;
  }
  // The ring also holds a split tile's sums.
  const size_t sums = SPLIT ? size_t((a.n + 31) / 32) * ((a.xrows + 31) / 32) * kStageTile : 0;
  a.ring = unsigned(std::max(q_ring_bytes(wrows, a.xrows, a.stages), sums));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = SPLIT ? dim3(unsigned(a.mtiles * a.ntiles * p.splits))
                      : dim3(unsigned(CG * std::min<long long>((long long)a.mtiles * a.ntiles, d->sms / CG)));
  cfg.blockDim = dim3(kQThreads);
  cfg.dynamicSmemBytes = std::max(kQMinSmem, a.ring + a.recv + kQFixed);
  cfg.stream = d->stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim = {unsigned(SPLIT ? p.splits : CG), 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = CG == 2 || SPLIT ? 2 : 1;
  cudaLaunchKernelEx(&cfg, k_gemm_q8<CG, SPLIT>, tw, tx, tout, tout16, a);
  return rt::launched("matmul_q8");
}

int gemm_q8(tb200_device* d, float* out, const tb200_q8* w, const tb200_q8* x) {
  QGemmArgs a{};
  a.sw = w->scales;
  a.sx = x->scales;
  a.out = out;
  a.T = int(x->rows);
  a.M = int(w->rows);
  a.K = int(w->cols);
  a.err = d->async_err_dev;
  a.tma_out = reinterpret_cast<uintptr_t>(out) % 16 == 0 && a.M % 4 == 0;
  // Pairs take fewer bytes from L2 but wait for one another: 1999 x 9728 x 2560 takes 43.8 us with
  // pairs and 47.8 without, 512 x 4096 x 1024 6.9 and 5.7.
  if (a.T >= 1024 && a.K >= 2048)
    return launch_gemm_q8<2, false>(d, a, plan_pair(a.M, (a.T + 2 * kTileM - 1) / (2 * kTileM), d->sms / 2), w, x);
  const QPlan p = plan_one(a.M, (a.K + kKB - 1) / kKB, a.T, d->sms);
  return p.splits > 1 ? launch_gemm_q8<1, true>(d, a, p, w, x) : launch_gemm_q8<1, false>(d, a, p, w, x);
}

}  // namespace

cudaError_t init_q8_kernels() {
  const auto most = cudaFuncAttributeMaxDynamicSharedMemorySize;
  cudaError_t e = cudaFuncSetAttribute(k_gemm_q8<1, false>, most, int(kQMaxSmem));
  if (e == cudaSuccess) e = cudaFuncSetAttribute(k_gemm_q8<1, true>, most, int(kQMaxSmem));
  if (e == cudaSuccess) e = cudaFuncSetAttribute(k_gemm_q8<2, false>, most, int(kQMaxSmem));
  return e;
}

}  // namespace tb

extern "C" {

int tb200_matmul_q8(tb200_device* d, tb200_buffer* out, const tb200_q8* w, const tb200_q8* x) {
  if (int rc = rt::use(d)) return rc;
  ARG_CHECK(out && w && x, "null argument");
  ARG_CHECK(rt::of(d, out, w, x), "matmul_q8: an operand was made on another device");
  ARG_CHECK(w->cols == x->cols, "matmul_q8: weight has " + std::to_string(w->cols) + " columns, input " +
                                    std::to_string(x->cols));
  ARG_CHECK(w->cols <= tb::kMaxCols, "matmul_q8: more than 131071 columns do not sum in 32 bits");
  ARG_CHECK(out->len == x->rows * w->rows, "matmul_q8: output holds " + std::to_string(out->len) + ", expected " +
                                               std::to_string(x->rows * w->rows));
  if (!x->rows || !w->rows) return TB200_OK;
  // Three to eight tokens over many weights keep the CUDA cores busy for longer than the weights take to arrive
  // (us there and on the tensor cores: four tokens, 2560 x 9728 8.4 and 9.4, 151936 x 1024 33.6 and 28.1; eight,
  // 1024 x 2048 2.1 and 4.9, 2560 x 4096 6.0 and 6.9, 9728 x 2560 9.9 and 7.9), but few channels make few tiles
  // (eight tokens, 1000 x 20000 7.2 and 12.3).
  const bool few = w->rows <= size_t(8) * d->sms;
  if (x->rows > 8 || (x->rows > 2 && !few && x->rows * w->rows * w->cols > size_t(128) << 20))
    return tb::gemm_q8(d, out->ptr, w, x);
  switch (x->rows) {
    case 1: tb::matvec_q8<1>(d, out->ptr, w, x); break;
    case 2: tb::matvec_q8<2>(d, out->ptr, w, x); break;
    case 3: tb::matvec_q8<3>(d, out->ptr, w, x); break;
    case 4: tb::matvec_q8<4>(d, out->ptr, w, x); break;
    case 5: tb::matvec_q8<5>(d, out->ptr, w, x); break;
    case 6: tb::matvec_q8<6>(d, out->ptr, w, x); break;
    case 7: tb::matvec_q8<7>(d, out->ptr, w, x); break;
    default: tb::matvec_q8<8>(d, out->ptr, w, x);
  }
  return rt::launched("matmul_q8");
}

}  // extern "C"
