// y = act(x W^T + bias) with x [M, K] and W [N, K] in e4m3 and one fp32 scale for each block of 128 along K
// (of every row of x; of every 128 rows of W):
//   y[m, n] = sum_c xs[m, c] ws[n / 128, c] sum_{k in block c} x[m, k] w[n, k]
// The inner sums run on the tensor cores (tcgen05.mma kind::f8f6f4, fp32 accumulators in TMEM); the scales
// differ from block to block, so every inner sum is taken out of TMEM, scaled and added in registers.
//
// A CTA holds 128 rows of x by 256 columns of sums; a pair of CTAs (a cluster, tcgen05 cta_group::2) shares a tile of 256
// rows, each loading half of W's 256 rows, and few tiles go to single CTAs.  The CTAs are persistent, one on an SM.  A
// step is one block of 128 along K, which is also one 128-byte swizzle row of the operands in shared memory:
//   warp 9      loads the step's operands by TMA into a ring
//   warp 10     copies the step's scales (128 of x, 2 of W) into a ring of their own, up to 16 steps ahead: read when they
//               are needed, they arrive later than the MMAs
//   warp 8      issues the step's four MMAs (K = 32 each) into one of two TMEM buffers of 256 columns
//   warps 0-7   two warpgroups, one for each block of 128 columns: thread = row, 128 fp32 sums in registers; they add the
//               scaled buffer of one step while the tensor core fills the other
// After the last step the sums get bias and activation and are rounded once; they leave through shared memory and
// TMA stores, which also clip the edges (16-byte stores from registers, 32 rows an instruction, cost a fifth of
// the whole time).  Or they become e4m3 rows again: a thread holds a whole block of its row.
//
// What bounds it: the MMAs alone take 533 cycles a step by pairs (595 by single CTAs; 512 is the tensor core's rate), the
// scaled sums bring that to about 700, and the tensor core waits for a tile's epilogue, which the summing warps do too: 4.5
// us a tile, 6.8 with GELU (9472 x K to 9728 over K: 0.41 us a step beside that).  The sums are 256 cycles of packed FMAs and
// the TMEM reads of two warps a scheduler, and what counted was keeping the rest out of their way: scales copied ahead, the next 16 columns loaded while the
// last ones are added, the buffer released before its last sums, arrivals without branches, the loop unrolled by
// four (853 cycles without these).  Four warpgroups of 64 columns run out of registers (855).  Over seconds the power
// limit sets the clock: 75,600 x 5120 x 15360 takes 5.57-5.73 ms (2.07-2.13 PFLOP/s) at about 1.4 GHz, a library product with
// one scale for everything 4.5-4.6 ms; 9450 x 5120 x 13824 takes 574-630 us (results in fp32 855, 16-bit ones off 16-byte
// words 1706: they leave lane by lane).  Few tiles of a long K axis go to the kernel for few rows, which splits it.
//
// Every wait on an mbarrier is bounded in time; when one gives up the CTA raises a flag in shared memory, all
// roles leave their loops, outstanding copies and MMAs are drained with bounded waits, TMEM is freed and
// *status is set.
#include <cstring>
#include <mutex>

#include "fp8_quant.cuh"
#include "sm100_ptx.cuh"

namespace xdit {
namespace {

constexpr int kThreads = 384;  // 8 summing warps, MMA warp, TMA warp, scale warp, 1 idle warp (full register-trading warpgroup)
constexpr int kSumWarps = 8;
constexpr int kBM = 128, kBN = 256, kBK = XDIT_FP8_BLOCK;
constexpr int kCols = 128;     // columns of a summing thread: those that share a scale of W
constexpr int kAhead = 16;     // steps whose scales are in shared memory or on their way
constexpr int kGroup = 4, kGroups = kAhead / kGroup;  // steps whose scales share a barrier
constexpr int kABytes = kBM * kBK;
constexpr int kWarpOut = 32 * kCols * 2;  // staging of a summing warp's results
constexpr int kScaleBytes = 576;          // 128 scales of x + 2 of w, padded
// Bytes of x in a band of row tiles, whose tiles are walked column by column: the band stays in L2 while W passes, and the
// fewer bands, the seldomer W passes (75,600 x 5120 x 15360: 10 MB 5.88 ms, 21 MB 5.75, 42 MB 5.83, 84 MB 6.35; 9450 x 13824 x
// 5120: 14 MB 663 us, 28 MB 648, 57 MB 658, 113 MB 686).
constexpr int64_t kBandBytes = 24 << 20;

template <bool PAIR> struct GemmLayout {
  static constexpr int kStages = PAIR ? 4 : 3;
  static constexpr int kBRows = PAIR ? kBN / 2 : kBN;        // rows of W that a CTA loads
  static constexpr int kStageBytes = kABytes + kBRows * kBK;
  static constexpr int kOutOff = kStages * kStageBytes;
  static constexpr int kBiasOff = kOutOff + kSumWarps * kWarpOut;   // [8 warps][128 columns]
  static constexpr int kScaleOff = kBiasOff + kSumWarps * kCols * 4;     // [kAhead]
  static constexpr int kBarOff = kScaleOff + kAhead * kScaleBytes;
  static constexpr int kNumBars = 2 * kStages + 4 + 1 + 2 * kGroups;
  static constexpr int kMiscOff = kBarOff + kNumBars * 8;
  static constexpr int kSmem = kMiscOff + 16 + 1024;  // with slack to align the base to 1024 bytes
};

struct alignas(64) GemmArgs {
  CUtensorMap tm_x, tm_w, tm_out;
  int32_t M, N, kb;        // kb: blocks along K
  int32_t mt, nt;          // tiles
  int32_t band;            // row tiles of a band
  int32_t splits;          // CTAs of a cluster that share the K axis of a tile (few rows)
  const float* xs;
  int64_t xs_srow, xs_skb;
  const float* ws;
  int64_t ws_snb, ws_skb;
  const void* bias;
  int32_t bias_dtype, act, out_dtype;
  void* out;
  int64_t out_srow;
  uint8_t* out_q;
  float* out_scale;
  int64_t out_scale_ld;
  int32_t wide;            // 16-byte stores are possible
  int32_t tma_out;         // the results leave through shared memory and tm_out
  int32_t* status;
  int32_t* status_host;
  uint32_t wait_limit_ns;
  int32_t selftest_stall;  // test aid: nothing is loaded, so the first waits run out
};

__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* tm, uint32_t bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(dst), "l"(tm), "r"(bar), "r"(c0), "r"(c1) : "memory");
}
// 32 lanes x 16 consecutive columns -> 16 registers per thread
#define XDIT_TMEM_LD16(a, taddr)                                                                                   \
  asm volatile(                                                                                                    \
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "                                                                     \
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"                              \
      : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3]), "=r"(a[4]), "=r"(a[5]), "=r"(a[6]), "=r"(a[7]), "=r"(a[8]),   \
        "=r"(a[9]), "=r"(a[10]), "=r"(a[11]), "=r"(a[12]), "=r"(a[13]), "=r"(a[14]), "=r"(a[15])                    \
      : "r"(taddr) : "memory")
// The same load by one CTA of a pair, whose bytes are counted on a barrier of either CTA (`bar`: its address in the cluster).
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap* tm, uint32_t bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(dst), "l"(tm), "r"(bar), "r"(c0), "r"(c1) : "memory");
}
__device__ __forceinline__ uint32_t map_to_cta(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ uint32_t cta_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Arrival on a barrier of a CTA of the cluster (`bar`: its address in the cluster).
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Arrival of the lanes that have `yes`, without a branch: one between a TMEM load and the sums that use it makes the
// compiler move registers.
template <bool CLUSTER>
__device__ __forceinline__ void mbar_arrive_if(uint32_t bar, uint32_t yes) {
  if constexpr (CLUSTER)
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %1, 0;\n\t@p mbarrier.arrive.shared::cluster.b64 _, [%0];\n\t}" ::"r"(bar), "r"(yes) : "memory");
  else
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %1, 0;\n\t@p mbarrier.arrive.shared::cta.b64 _, [%0];\n\t}" ::"r"(bar), "r"(yes) : "memory");
}
// Completion of the MMAs issued so far, on the same barrier of both CTAs of a pair.
__device__ __forceinline__ void tc_commit_pair(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3) : "memory");
}
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* tm, uint32_t src, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(tm), "r"(src), "r"(c0), "r"(c1) : "memory");
}
__device__ __forceinline__ void st_shared16(uint32_t at, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
// acc += s * p for the pair of columns (acc0, acc1)
__device__ __forceinline__ void fma_pair(float& acc0, float& acc1, uint32_t p0, uint32_t p1, uint64_t s2) {
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 y, {%2, %3};\n\tfma.rn.f32x2 x, y, %4, x;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "+f"(acc0), "+f"(acc1) : "r"(p0), "r"(p1), "l"(s2));
}
__device__ __forceinline__ uint32_t pack16(int dtype, float lo, float hi) {
  if (dtype == XDIT_BF16) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  }
  __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
template <bool PAIR = false>
__device__ __forceinline__ void mma_f8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  if constexpr (PAIR)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
}
__device__ __forceinline__ float load_any(const void* p, int dtype, int64_t i) {
  if (dtype == XDIT_F32) return __ldg(reinterpret_cast<const float*>(p) + i);
  if (dtype == XDIT_BF16) return __bfloat162float(__ldg(reinterpret_cast<const __nv_bfloat16*>(p) + i));
  return __half2float(__ldg(reinterpret_cast<const __half*>(p) + i));
}
__device__ __forceinline__ void store_any(void* p, int dtype, int64_t i, float x) {
  if (dtype == XDIT_F32) reinterpret_cast<float*>(p)[i] = x;
  else if (dtype == XDIT_BF16) reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(x);
  else reinterpret_cast<__half*>(p)[i] = __float2half_rn(x);
}
__device__ __forceinline__ uint64_t f2_mul(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// x/2 (1 + tanh u) = x / (1 + exp(-2u)) with u = sqrt(2/pi) (x + 0.044715 x^3), for two values: the polynomial
// -2u log2(e) on packed pairs, then base-2 exponentials and reciprocals (2^-22 off).
__device__ __forceinline__ void gelu_tanh2(float& x0, float& x1) {
  constexpr float k1 = -2.f * 0.7978845608028654f * 1.4426950408889634f, k3 = k1 * 0.044715f;
  const uint64_t x = f2_pack(x0, x1);
  const uint64_t z = f2_mul(x, f2_fma(f2_mul(x, x), f2_pack(k3, k3), f2_pack(k1, k1)));
  float z0, z1;
  f2_unpack(z, z0, z1);
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(z0));
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(z1));
  z0 += 1.f;
  z1 += 1.f;
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(z0));
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(z1));
  x0 *= z0;
  x1 *= z1;
}
// A CTA whose wait gave up tells the later launches and the host.
__device__ __forceinline__ void report(const GemmArgs& a, volatile int* abort_flag) {
  if (threadIdx.x == 0 && *abort_flag > 0) {
    if (a.status) atomicCAS(a.status, 0, *abort_flag);
    if (a.status_host) {  // host-visible copy, read by the next call without a synchronise
      *reinterpret_cast<volatile int32_t*>(a.status_host) = *abort_flag;
      __threadfence_system();
    }
  }
}
// A launch with quantising may start before the kernel that quantises x has ended.  Every CTA waits for that end, one that
// skips its work too: what comes next on the stream is ordered behind this kernel alone, and may be given the memory that
// the quantised rows are written to.
__device__ __forceinline__ void wait_for_quantise() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// Tile t: its row and column of tiles.
__device__ __forceinline__ void tile_at(const GemmArgs& a, int t, int& m, int& n) {
  const int band = t / (a.band * a.nt), rem = t - band * a.band * a.nt;
  const int high = min(a.band, a.mt - band * a.band);
  n = rem / high;
  m = band * a.band + rem - n * high;
}

template <bool PAIR>
__global__ void __launch_bounds__(kThreads, 1) fp8_gemm_kernel(const __grid_constant__ GemmArgs a) {
  using L = GemmLayout<PAIR>;
  constexpr int kStages = L::kStages, kRows = PAIR ? 2 * kBM : kBM;  // rows of a tile
  extern __shared__ unsigned char smem_dyn[];
  const uint32_t raw = smem_u32(smem_dyn), base = (raw + 1023u) & ~1023u;
  unsigned char* base_ptr = smem_dyn + (base - raw);
  const uint32_t bar0 = base + L::kBarOff;
  auto bar_full = [&](int s) { return bar0 + 8u * s; };
  auto bar_empty = [&](int s) { return bar0 + 8u * (kStages + s); };
  auto bar_tfull = [&](int s) { return bar0 + 8u * (2 * kStages + s); };
  auto bar_tempty = [&](int s) { return bar0 + 8u * (2 * kStages + 2 + s); };
  const uint32_t bar_drain = bar0 + 8u * (2 * kStages + 4);
  auto bar_sfull = [&](int s) { return bar0 + 8u * (2 * kStages + 5 + s); };
  auto bar_sempty = [&](int s) { return bar0 + 8u * (2 * kStages + 5 + kGroups + s); };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(base_ptr + L::kMiscOff);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(base_ptr + L::kMiscOff + 4);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tiles = a.mt * a.nt;
  // A pair of CTAs (a cluster) shares a tile: each holds its 128 rows of x and of the sums, and half of W's rows; the
  // first one, `rank` 0, issues the MMAs of both.
  const int rank = PAIR ? (int)cta_rank() : 0;
  const int tile0 = PAIR ? blockIdx.x / 2 : blockIdx.x, tile_step = PAIR ? gridDim.x / 2 : gridDim.x;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) { mbar_init(bar_full(s), 1); mbar_init(bar_empty(s), 1); }
    for (int s = 0; s < 2; ++s) { mbar_init(bar_tfull(s), 1); mbar_init(bar_tempty(s), PAIR ? 2 * kSumWarps : kSumWarps); }
    for (int s = 0; s < kGroups; ++s) { mbar_init(bar_sfull(s), 32); mbar_init(bar_sempty(s), kSumWarps); }
    mbar_init(bar_drain, 1);
    *abort_flag = status_is_set(a.status) ? -1 : 0;  // -1: skip all work (an earlier failure is pending)
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 8) {
    if constexpr (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  bool skip = *abort_flag != 0;  // same value for every thread: written before the barrier above
  if constexpr (PAIR) {
    // the other CTA's barriers are ready behind this, and both skip where one has seen a failure
    cluster_sync();
    uint32_t other;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(other) : "r"(map_to_cta(smem_u32(const_cast<int*>(abort_flag)), rank ^ 1)) : "memory");
    skip |= other != 0;
    cluster_sync();  // neither changes its flag before both have read them
  }

  if (skip) {
    // nothing to do: fall through to the teardown, which frees TMEM
    wait_for_quantise();
  } else if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");  // per scheduler 2 x 232 + 40 = 3 x 168, what the launch holds
    if (warp == 9) {
      // ======================= TMA producer =======================
      if (lane == 0) {
        wait_for_quantise();  // x is complete from here on
        int issued = 0;
        bool ok = a.selftest_stall == 0;
        for (int t = tile0; t < tiles && ok; t += tile_step) {
          int m, n;
          tile_at(a, t, m, n);
          for (int c = 0; c < a.kb; ++c) {
            const int st = issued % kStages, turn = issued / kStages;
            if (turn > 0) ok = mbar_wait(bar_empty(st), (turn - 1) & 1, abort_flag, a.wait_limit_ns, 100 + st);
            if (!ok) break;
            const uint32_t to = base + st * L::kStageBytes;
            if constexpr (PAIR) {  // both CTAs' bytes count on the first one's barrier
              if (rank == 0) mbar_arrive_expect_tx(bar_full(st), 2 * L::kStageBytes);
              const uint32_t full = map_to_cta(bar_full(st), 0);
              tma_load_2d_pair(to, &a.tm_x, full, c * kBK, m * kRows + rank * kBM);
              tma_load_2d_pair(to + kABytes, &a.tm_w, full, c * kBK, n * kBN + rank * L::kBRows);
            } else {
              mbar_arrive_expect_tx(bar_full(st), L::kStageBytes);
              tma_load_2d(to, &a.tm_x, bar_full(st), c * kBK, m * kBM);
              tma_load_2d(to + kABytes, &a.tm_w, bar_full(st), c * kBK, n * kBN);
            }
            ++issued;
          }
        }
        // the MMAs report the last stages' release (of a pair, to both CTAs): none may leave before that has arrived
        for (int i = issued > kStages ? issued - kStages : 0; i < issued && ok; ++i)
          ok = mbar_wait(bar_empty(i % kStages), (i / kStages) & 1, abort_flag, a.wait_limit_ns, 110);
        if (!ok) {
          // drain: every armed stage must have received its bytes before the CTA may leave (a pair: before either leaves)
          // (the second CTA's bytes count on the first one's barriers, which it cannot watch: it leaves them a thousand times
          // the time that a load takes)
          if (rank) for (int it = 0; it < (1 << 14); ++it) __nanosleep(128);
          for (int i = rank ? issued : issued > kStages ? issued - kStages : 0; i < issued; ++i)
            for (int it = 0; it < (1 << 20) && !mbar_try_wait(bar_full(i % kStages), (i / kStages) & 1); ++it) __nanosleep(64);
        }
      }
    } else if (warp == 10) {
      // ======================= scales: each lane the rows lane, lane + 32, ... of the tile =======================
      // A load from L2 takes longer than a step, so they are copied asynchronously, up to kAhead steps ahead.
      wait_for_quantise();
      int step = 0;
      bool ok = true;
      for (int t = tile0; t < tiles && ok; t += tile_step) {
        int m, n;
        tile_at(a, t, m, n);
        const float* src[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = m * kRows + rank * kBM + 32 * i + lane;  // rows and columns behind the end take any scale
          src[i] = a.xs + (int64_t)(row < a.M ? row : 0) * a.xs_srow;
        }
        const int nb = n * (kBN / kBK) + (lane & 1);
        const float* w = a.ws + (int64_t)(nb * kBK < a.N ? nb : 0) * a.ws_snb;
        for (int c = 0; c < a.kb; ++c, ++step) {
          const int slot = step % kAhead, turn = step / kAhead, group = slot / kGroup;
          if (turn > 0 && step % kGroup == 0) ok = __all_sync(0xffffffffu, mbar_wait(bar_sempty(group), (turn - 1) & 1, abort_flag, a.wait_limit_ns, 320));
          if (!ok) break;
          const uint32_t at = base + L::kScaleOff + slot * kScaleBytes + lane * 4;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(at + 128 * i), "l"(src[i]) : "memory");
            src[i] += a.xs_skb;
          }
          if (lane < 2) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(at + 512), "l"(w) : "memory");
          w += a.ws_skb;
          if (step % kGroup == kGroup - 1)
            asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar_sfull(group)) : "memory");
        }
      }
      if (step % kGroup)  // the last group is not full
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar_sfull(step % kAhead / kGroup)) : "memory");
      asm volatile("cp.async.wait_all;" ::: "memory");
    } else if (warp == 8 && rank == 0) {
      // ======================= MMA issuer (the warp runs converged, one elected lane issues) =======================
      const bool leader = elect_one();
      const uint32_t tmem_u = __shfl_sync(0xffffffffu, tmem_base, 0);
      const uint32_t idesc = (1u << 4) | ((uint32_t)(kBN >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);  // e4m3 x e4m3 -> fp32
      bool ok = true;
      int step = 0;
      auto wait_all = [&](uint32_t bar, uint32_t parity, int code) {
        return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, a.wait_limit_ns, code));
      };
      for (int t = tile0; t < tiles && ok; t += tile_step) {
        for (int c = 0; c < a.kb; ++c, ++step) {
          const int st = step % kStages, buf = step & 1;
          ok = wait_all(bar_full(st), (step / kStages) & 1, 210 + st);
          if (ok && step >= 2) ok = wait_all(bar_tempty(buf), ((step >> 1) - 1) & 1, 200 + buf);
          if (!ok) break;
          tc_fence_after();
          if (leader) {
            const uint64_t da = desc_kmajor(base + st * L::kStageBytes), db = desc_kmajor(base + st * L::kStageBytes + kABytes);
#pragma unroll
            for (int k = 0; k < kBK / 32; ++k) mma_f8<PAIR>(tmem_u + buf * kBN, da + 2 * k, db + 2 * k, idesc, k > 0);
            if constexpr (PAIR) {
              tc_commit_pair(bar_tfull(buf));
              tc_commit_pair(bar_empty(st));
            } else {
              tc_commit(bar_tfull(buf));
              tc_commit(bar_empty(st));
            }
          }
        }
      }
      if (!ok) {
        // drain the tensor pipe before TMEM is released
        if (leader) {
          if constexpr (PAIR) tc_commit_pair(bar_drain);
          else tc_commit(bar_drain);
        }
        if (lane == 0)
          for (int it = 0; it < (1 << 20) && !mbar_try_wait(bar_drain, 0); ++it) __nanosleep(64);
        __syncwarp();
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
    // ======================= scaled sums + epilogue =======================
    const int group = warp >> 2;  // columns [128 group, 128 group + 128) of the tile
    const uint32_t taddr = tmem_base + ((uint32_t)((warp & 3) * 32) << 16) + group * kCols;
    const uint32_t scale_x = base + L::kScaleOff + ((warp & 3) * 32 + lane) * 4, scale_w = base + L::kScaleOff + 512 + group * 4;
    const uint32_t tempty_at = PAIR ? map_to_cta(bar_tempty(0), 0) : bar_tempty(0);
    bool ok = true;
    int step = 0;
    for (int t = tile0; t < tiles && ok; t += tile_step) {
      if (a.bias) {
        int m, n;
        tile_at(a, t, m, n);
        const int col0 = n * kBN + group * kCols;
        float* bias = reinterpret_cast<float*>(base_ptr + L::kBiasOff) + warp * kCols;
        __syncwarp();
#pragma unroll
        for (int i = 0; i < kCols; i += 32)
          bias[i + lane] = col0 + i + lane < a.N ? load_any(a.bias, a.bias_dtype, col0 + i + lane) : 0.f;
        __syncwarp();
      }
      float acc[kCols];
#pragma unroll
      for (int i = 0; i < kCols; ++i) acc[i] = 0;
#pragma unroll 4
      for (int c = 0; c < a.kb; ++c, ++step) {
        const int buf = step & 1, slot = step % kAhead;
        // no way out of this loop: with one, the compiler copies all sums in every step.  After a wait that gave
        // up, the others return at once.
        if (step % kGroup == 0) ok &= mbar_wait(bar_sfull(slot / kGroup), (step / kAhead) & 1, abort_flag, a.wait_limit_ns, 310);
        ok &= mbar_wait(bar_tfull(buf), (step >> 1) & 1, abort_flag, a.wait_limit_ns, 300 + buf);
        __syncwarp();
        tc_fence_after();
        const uint32_t tb = taddr + buf * kBN;
        uint32_t p[2][16];
        XDIT_TMEM_LD16(p[0], tb);
        float sx, sw;
        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(sx) : "r"(scale_x + slot * kScaleBytes) : "memory");
        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(sw) : "r"(scale_w + slot * kScaleBytes) : "memory");
        const uint64_t s2 = f2_pack(sx * sw, sx * sw);
        tmem_wait_ld();
#pragma unroll
        for (int q = 0; q < kCols; q += 16) {
          const int h = (q >> 4) & 1;
          if (q + 16 < kCols) XDIT_TMEM_LD16(p[h ^ 1], tb + q + 16);
#pragma unroll
          for (int i = 0; i < 16; i += 2) fma_pair(acc[q + i], acc[q + i + 1], p[h][i], p[h][i + 1], s2);
          if (q + 16 < kCols) tmem_wait_ld();
          if (q + 32 == kCols) {  // the buffer has been read
            tc_fence_before();
            __syncwarp();
            mbar_arrive_if<PAIR>(tempty_at + 8u * buf, lane == 0);
            mbar_arrive_if<false>(bar_sempty(slot / kGroup), lane == 0 && step % kGroup == kGroup - 1);
          }
        }
      }
      ok = __all_sync(0xffffffffu, ok);
      int m, n;
      tile_at(a, t, m, n);
      const int row0 = m * kRows + rank * kBM + (warp & 3) * 32, col0 = n * kBN + group * kCols;
      const int64_t row = row0 + lane;
      const bool live = ok && row < a.M && col0 < a.N;
      const uint32_t stage = base + L::kOutOff + warp * kWarpOut;
      if (a.bias) {
        const float* bias = reinterpret_cast<const float*>(base_ptr + L::kBiasOff) + warp * kCols;
#pragma unroll
        for (int i = 0; i < kCols; i += 4) {
          const float4 v = *reinterpret_cast<const float4*>(bias + i);
          acc[i] += v.x; acc[i + 1] += v.y; acc[i + 2] += v.z; acc[i + 3] += v.w;
        }
      }
      if (a.act == XDIT_ACT_GELU_TANH) {
#pragma unroll
        for (int i = 0; i < kCols; i += 2) gelu_tanh2(acc[i], acc[i + 1]);
      }
      if (a.tma_out) {  // the last tile's results have left the staging buffer
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        __syncwarp();
      }
      if (a.out_q) {
        // the thread holds a whole block of its row; columns behind the end were loaded as zeros and are zeros still
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < kCols; i += 2) top = amax_nan(top, acc[i], acc[i + 1]);
        float inv;
        const float sc = block_scale(top, inv);
        if (live) a.out_scale[(col0 / kBlock) * a.out_scale_ld + row] = sc;
#pragma unroll
        for (int i = 0; i < kCols; i += 16) {
          uint4 w;
          w.x = pack_e4m3(acc[i] * inv, acc[i + 1] * inv, acc[i + 2] * inv, acc[i + 3] * inv);
          w.y = pack_e4m3(acc[i + 4] * inv, acc[i + 5] * inv, acc[i + 6] * inv, acc[i + 7] * inv);
          w.z = pack_e4m3(acc[i + 8] * inv, acc[i + 9] * inv, acc[i + 10] * inv, acc[i + 11] * inv);
          w.w = pack_e4m3(acc[i + 12] * inv, acc[i + 13] * inv, acc[i + 14] * inv, acc[i + 15] * inv);
          st_shared16(stage + lane * 128 + (((i >> 4) ^ (lane & 7)) << 4), w);  // 128-byte swizzle
        }
      } else if (a.tma_out) {
#pragma unroll
        for (int i = 0; i < kCols; i += 8) {  // two boxes of 64 columns
          uint4 w;
          w.x = pack16(a.out_dtype, acc[i], acc[i + 1]);
          w.y = pack16(a.out_dtype, acc[i + 2], acc[i + 3]);
          w.z = pack16(a.out_dtype, acc[i + 4], acc[i + 5]);
          w.w = pack16(a.out_dtype, acc[i + 6], acc[i + 7]);
          st_shared16(stage + (i >> 6) * 4096 + lane * 128 + ((((i & 63) >> 3) ^ (lane & 7)) << 4), w);  // 128-byte swizzle
        }
      } else if (live) {
        const int64_t o = row * a.out_srow + col0;
#pragma unroll
        for (int i = 0; i < kCols; i += 4) {
          if (a.wide && a.out_dtype == XDIT_F32 && col0 + i + 4 <= a.N) {
            *reinterpret_cast<float4*>(reinterpret_cast<float*>(a.out) + o + i) = make_float4(acc[i], acc[i + 1], acc[i + 2], acc[i + 3]);
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (col0 + i + j < a.N) store_any(a.out, a.out_dtype, o + i + j, acc[i + j]);
          }
        }
      }
      if (a.tma_out) {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0 && ok && row0 < a.M) {  // what lies behind the end of a row or column is not written
          if (col0 < a.N) tma_store_2d(&a.tm_out, stage, col0, row0);
          if (!a.out_q && col0 + 64 < a.N) tma_store_2d(&a.tm_out, stage + 4096, col0 + 64, row0);
          asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
      }
    }
    if (a.tma_out && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }

  // ---------------- teardown ----------------
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync();  // neither leaves while the other may still reach its barriers or TMEM
  if (warp == 8) {
    tc_fence_after();
    if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512) : "memory");
  }
  report(a, abort_flag);
}

// ---------------------------------------------------------------------------------------------------
// Few rows of x: the weight's bytes bound the time, so the operands change places.  A tile is 128 rows of W (the
// M side of the MMA) by NB rows of x, small enough for two CTAs on an SM, with a deep ring of W in flight; a thread
// holds NB sums of its row of W.  When there are fewer tiles than SMs can use, the K axis is split over the CTAs of a
// cluster: each leaves its sums in shared memory, and each then adds the cluster's sums, in their order, for a share of the
// rows of x -- no scratch in global memory, and the same result every time.
//   warps 0-3  scaled sums + epilogue      warp 4  MMA      warp 5  TMA      warp 6  scales
// The kernel may start while the one that quantises x is still running (griddepcontrol): W is loaded at once, x and
// its scales after that kernel's end.
// Two rows by 30,720 x 5120 (157 MB of W): 28-29 us in a stream of calls, 5.4-5.6 TB/s or 0.83-0.86 of a copy; by the kernel
// above 50.5 us.  Small products are bound by the chain of one step after another: about 10 us a call in the end.
constexpr int kRowsThreads = 224;
constexpr int kMaxSplits = 8;  // the largest portable cluster

template <int NB> struct RowsLayout {
  static constexpr int kStages = NB <= 16 ? 6 : NB <= 32 ? 5 : 4;
  static constexpr int kStageBytes = kABytes + NB * kBK;
  static constexpr int kSlot = NB * 4 + 16;                   // scales of a step: NB of x, one of W
  static constexpr int kAhead = 8, kGroup = 4, kGroups = kAhead / kGroup;
  static constexpr int kScaleOff = kStages * kStageBytes;
  static constexpr int kTopOff = kScaleOff + kAhead * kSlot;  // [4 warps][NB] largest magnitudes
  static constexpr int kBarOff = kTopOff + 4 * NB * 4;
  static constexpr int kNumBars = 2 * kStages + 4 + 1 + 2 * kGroups;
  static constexpr int kMiscOff = kBarOff + kNumBars * 8;
  static constexpr int kSmem = kMiscOff + 16 + 1024;
  static_assert(kStages * kStageBytes >= 128 * NB * 4, "the ring holds the sums that a cluster exchanges");
};

__device__ __forceinline__ float4 load_cluster(uint32_t addr, uint32_t rank) {
  float4 v;
  asm volatile(
      "{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %4, %5;\n\t"
      "ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [a];\n\t}"
      : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr), "r"(rank) : "memory");
  return v;
}

template <int NB>
__global__ void __launch_bounds__(kRowsThreads, 2) fp8_rows_kernel(const __grid_constant__ GemmArgs a) {
  using L = RowsLayout<NB>;
  constexpr int kStages = L::kStages;
  extern __shared__ unsigned char smem_dyn[];
  const uint32_t raw = smem_u32(smem_dyn), base = (raw + 1023u) & ~1023u;
  unsigned char* base_ptr = smem_dyn + (base - raw);
  const uint32_t bar0 = base + L::kBarOff;
  auto bar_full = [&](int s) { return bar0 + 8u * s; };
  auto bar_empty = [&](int s) { return bar0 + 8u * (kStages + s); };
  auto bar_tfull = [&](int s) { return bar0 + 8u * (2 * kStages + s); };
  auto bar_tempty = [&](int s) { return bar0 + 8u * (2 * kStages + 2 + s); };
  const uint32_t bar_drain = bar0 + 8u * (2 * kStages + 4);
  auto bar_sfull = [&](int s) { return bar0 + 8u * (2 * kStages + 5 + s); };
  auto bar_sempty = [&](int s) { return bar0 + 8u * (2 * kStages + 5 + L::kGroups + s); };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(base_ptr + L::kMiscOff);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(base_ptr + L::kMiscOff + 4);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kTmem = 2 * NB < 32 ? 32 : 2 * NB;
  // blockIdx.x = (tile of W) * splits + split, blockIdx.y = tile of x
  const int split = blockIdx.x % a.splits, n0 = (blockIdx.x / a.splits) * 128, m0 = blockIdx.y * NB;
  const int c0 = (int)((int64_t)split * a.kb / a.splits), steps = (int)((int64_t)(split + 1) * a.kb / a.splits) - c0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) { mbar_init(bar_full(s), 1); mbar_init(bar_empty(s), 1); }
    for (int s = 0; s < 2; ++s) { mbar_init(bar_tfull(s), 1); mbar_init(bar_tempty(s), 4); }
    for (int s = 0; s < L::kGroups; ++s) { mbar_init(bar_sfull(s), 32); mbar_init(bar_sempty(s), 4); }
    mbar_init(bar_drain, 1);
    *abort_flag = status_is_set(a.status) ? -1 : 0;  // -1: skip all work (an earlier failure is pending)
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 4) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(kTmem) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const bool skip = *abort_flag != 0;  // same value for every thread: written before the barrier above
  bool ok = !skip;
  float acc[NB];
#pragma unroll
  for (int i = 0; i < NB; ++i) acc[i] = 0.f;

  if (skip) {
    // nothing to do: fall through to the teardown, which frees TMEM
    wait_for_quantise();
  } else if (warp == 5) {
    // ======================= TMA producer =======================
    if (lane == 0) {
      auto load_w = [&](int i) {
        mbar_arrive_expect_tx(bar_full(i % kStages), L::kStageBytes);
        tma_load_2d(base + (i % kStages) * L::kStageBytes, &a.tm_w, bar_full(i % kStages), (c0 + i) * kBK, n0);
      };
      auto load_x = [&](int i) {
        tma_load_2d(base + (i % kStages) * L::kStageBytes + kABytes, &a.tm_x, bar_full(i % kStages), (c0 + i) * kBK, m0);
      };
      const int first = a.selftest_stall ? 0 : min(steps, kStages);
      for (int i = 0; i < first; ++i) load_w(i);
      wait_for_quantise();  // x is complete from here on
      for (int i = 0; i < first; ++i) load_x(i);
      int issued = first;
      ok = a.selftest_stall == 0;
      for (; ok && issued < steps; ++issued) {
        ok = mbar_wait(bar_empty(issued % kStages), (issued / kStages - 1) & 1, abort_flag, a.wait_limit_ns, 100);
        if (!ok) break;
        load_w(issued);
        load_x(issued);
      }
      // the MMAs report the last stages' release: the CTA may not leave before that has arrived
      for (int i = issued > kStages ? issued - kStages : 0; i < issued && ok; ++i)
        ok = mbar_wait(bar_empty(i % kStages), (i / kStages) & 1, abort_flag, a.wait_limit_ns, 110);
      if (!ok) {
        // drain: every armed stage must have received its bytes before the CTA may leave
        for (int i = issued > kStages ? issued - kStages : 0; i < issued; ++i)
          for (int it = 0; it < (1 << 20) && !mbar_try_wait(bar_full(i % kStages), (i / kStages) & 1); ++it) __nanosleep(64);
      }
    }
  } else if (warp == 6) {
    // ======================= scales =======================
    wait_for_quantise();
    constexpr int kPer = (NB + 31) / 32;
    const float* src[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int row = m0 + 32 * i + lane;  // rows behind the end take any scale
      src[i] = a.xs + (int64_t)(row < a.M ? row : 0) * a.xs_srow + c0 * a.xs_skb;
    }
    const float* w = a.ws + (n0 / kBK) * a.ws_snb + c0 * a.ws_skb;
    int step = 0;
    for (; step < steps; ++step) {
      const int slot = step % L::kAhead, turn = step / L::kAhead;
      if (turn > 0 && step % L::kGroup == 0)
        ok = __all_sync(0xffffffffu, mbar_wait(bar_sempty(slot / L::kGroup), (turn - 1) & 1, abort_flag, a.wait_limit_ns, 320));
      if (!ok) break;
      const uint32_t at = base + L::kScaleOff + slot * L::kSlot;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        if (32 * i + lane < NB)
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(at + (32 * i + lane) * 4), "l"(src[i]) : "memory");
        src[i] += a.xs_skb;
      }
      if (lane == 0) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(at + NB * 4), "l"(w) : "memory");
      w += a.ws_skb;
      if (step % L::kGroup == L::kGroup - 1 || step == steps - 1)
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar_sfull(slot / L::kGroup)) : "memory");
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else if (warp == 4) {
    // ======================= MMA issuer (the warp runs converged, one elected lane issues) =======================
    const bool leader = elect_one();
    const uint32_t tmem_u = __shfl_sync(0xffffffffu, tmem_base, 0);
    const uint32_t idesc = (1u << 4) | ((uint32_t)(NB >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);  // e4m3 x e4m3 -> fp32
    auto wait_all = [&](uint32_t bar, uint32_t parity, int code) {
      return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, a.wait_limit_ns, code));
    };
    for (int step = 0; step < steps; ++step) {
      const int st = step % kStages, buf = step & 1;
      ok = wait_all(bar_full(st), (step / kStages) & 1, 210 + st);
      if (ok && step >= 2) ok = wait_all(bar_tempty(buf), ((step >> 1) - 1) & 1, 200 + buf);
      if (!ok) break;
      tc_fence_after();
      if (leader) {
        const uint64_t dw = desc_kmajor(base + st * L::kStageBytes), dx = desc_kmajor(base + st * L::kStageBytes + kABytes);
#pragma unroll
        for (int k = 0; k < kBK / 32; ++k) mma_f8(tmem_u + buf * NB, dw + 2 * k, dx + 2 * k, idesc, k > 0);
        tc_commit(bar_tfull(buf));
        tc_commit(bar_empty(st));
      }
    }
    if (!ok) {
      // drain the tensor pipe before TMEM is released
      if (leader) tc_commit(bar_drain);
      if (lane == 0)
        for (int it = 0; it < (1 << 20) && !mbar_try_wait(bar_drain, 0); ++it) __nanosleep(64);
      __syncwarp();
    }
  } else if (warp < 4) {
    // ======================= scaled sums =======================
    const uint32_t taddr = tmem_base + ((uint32_t)(warp * 32) << 16);
#pragma unroll 1
    for (int step = 0; step < steps; ++step) {
      const int buf = step & 1, slot = step % L::kAhead;
      if (step % L::kGroup == 0) ok &= mbar_wait(bar_sfull(slot / L::kGroup), (step / L::kAhead) & 1, abort_flag, a.wait_limit_ns, 310);
      ok &= mbar_wait(bar_tfull(buf), (step >> 1) & 1, abort_flag, a.wait_limit_ns, 300 + buf);
      __syncwarp();
      tc_fence_after();
      const float* scales = reinterpret_cast<const float*>(base_ptr + L::kScaleOff + slot * L::kSlot);
      const uint64_t sw = f2_pack(scales[NB], scales[NB]);
      uint32_t p[2][16];
      XDIT_TMEM_LD16(p[0], taddr + buf * NB);
      tmem_wait_ld();
#pragma unroll
      for (int q = 0; q < NB; q += 16) {
        const int h = (q >> 4) & 1;
        if (q + 16 < NB) XDIT_TMEM_LD16(p[h ^ 1], taddr + buf * NB + q + 16);  // while these are added
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          const float4 sx = *reinterpret_cast<const float4*>(scales + q + i);
          fma_pair(acc[q + i], acc[q + i + 1], p[h][i], p[h][i + 1], f2_mul(f2_pack(sx.x, sx.y), sw));
          fma_pair(acc[q + i + 2], acc[q + i + 3], p[h][i + 2], p[h][i + 3], f2_mul(f2_pack(sx.z, sx.w), sw));
        }
        if (q + 16 < NB) tmem_wait_ld();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(bar_tempty(buf));
        if (step % L::kGroup == L::kGroup - 1) mbar_arrive(bar_sempty(slot / L::kGroup));
      }
    }
    ok = __all_sync(0xffffffffu, ok);
  }

  // ======================= epilogue =======================
  // The sums go to shared memory, [128 rows of W][NB], where the ring was: every MMA has read it by now, for the summing
  // warps have waited for all of them.  Rows [first, last) of the tile of x are this CTA's (without a split all of them):
  // it adds the cluster's sums of these, and nobody else reads its own ones, which take the results.  (Short loops, not
  // unrolled ones on the registers: with 64 rows the code that runs once cost 3 us more.)
  const int share = NB / a.splits, first = split * share, last = min(first + share, a.M - m0);
  const int n = n0 + warp * 32 + lane;
  const uint32_t mine = base + (warp * 32 + lane) * (NB * 4);
  auto place = [&](int i) { return (uint32_t)((i + 4 * lane) & (NB - 1)) * 4; };  // rotated: neighbours use other banks
  if (warp < 4) {
#pragma unroll
    for (int i = 0; i < NB; i += 4)
      asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(mine + place(i)), "f"(acc[i]), "f"(acc[i + 1]), "f"(acc[i + 2]), "f"(acc[i + 3]) : "memory");
  }
  if (a.splits > 1) cluster_sync();
  float* tops = reinterpret_cast<float*>(base_ptr + L::kTopOff);
  if (warp < 4) {
    const float bias = a.bias && n < a.N ? load_any(a.bias, a.bias_dtype, n) : 0.f;
    const int es = a.out_dtype == XDIT_F32 ? 4 : 2;
    const int64_t row_bytes = a.out_srow * es;
    char* o = reinterpret_cast<char*>(a.out) + (m0 + (first & ~3)) * row_bytes + (int64_t)n * es;
    const bool write = ok && n < a.N;
#pragma unroll 1
    for (int i = first & ~3; i < last; i += 4) {
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      float4 u[kMaxSplits];  // all on their way before the first is added: a load from another SM takes long
#pragma unroll
      for (int c = 0; c < kMaxSplits; ++c)
        if (c < a.splits) u[c] = a.splits > 1 ? load_cluster(mine + place(i), c) : *reinterpret_cast<const float4*>(base_ptr + (mine - base) + place(i));
#pragma unroll
      for (int c = 0; c < kMaxSplits; ++c)
        if (c < a.splits) { v.x += u[c].x; v.y += u[c].y; v.z += u[c].z; v.w += u[c].w; }
      float y[4] = {v.x + bias, v.y + bias, v.z + bias, v.w + bias};
      if (a.act == XDIT_ACT_GELU_TANH) { gelu_tanh2(y[0], y[1]); gelu_tanh2(y[2], y[3]); }
      if (a.out_q) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {  // a NaN's bits are above an infinity's
          const uint32_t top = __reduce_max_sync(0xffffffffu, n < a.N ? __float_as_uint(fabsf(y[j])) : 0u);
          if (lane == 0) tops[warp * NB + i + j] = __uint_as_float(top);
        }
        // rows of another CTA's share are left alone: it may be reading them
        if (i >= first && i + 4 <= first + share) {
          asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(mine + place(i)), "f"(y[0]), "f"(y[1]), "f"(y[2]), "f"(y[3]) : "memory");
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (i + j >= first && i + j < last)
              asm volatile("st.shared.f32 [%0], %1;" ::"r"(mine + place(i) + 4 * j), "f"(y[j]) : "memory");
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j, o += row_bytes) {
          if (!write || i + j < first || i + j >= last) continue;
          if (es == 4) {
            *reinterpret_cast<float*>(o) = y[j];
          } else {
            const uint32_t w = pack16(a.out_dtype, y[j], 0.f);
            *reinterpret_cast<uint16_t*>(o) = (uint16_t)w;
          }
        }
      }
    }
  }
  if (a.splits > 1) cluster_sync();  // nobody leaves while its sums are being read
  if (a.out_q) {
    // the tile's 128 columns of the result are one block: its rows' largest magnitudes over the four warps
    __syncthreads();
    if (warp < 4 && ok) {
#pragma unroll 1
      for (int i = first; i < last; ++i) {
        float inv, y;
        const float top = amax_nan(amax_nan(tops[i], tops[NB + i], tops[2 * NB + i]), tops[3 * NB + i]);
        const float sc = block_scale(top, inv);
        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(y) : "r"(mine + place(i & ~3) + 4 * (i & 3)) : "memory");
        const int64_t m = m0 + i;
        if (n < a.N) a.out_q[m * a.N + n] = (uint8_t)pack_e4m3(y * inv, 0.f, 0.f, 0.f);
        if (threadIdx.x == 0) a.out_scale[(n0 / kBlock) * a.out_scale_ld + m] = sc;
      }
    }
  }

  // ---------------- teardown ----------------
  tc_fence_before();
  __syncthreads();
  if (warp == 4) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmem) : "memory");
  }
  report(a, abort_flag);
}

// Map of a row-major matrix of `type`: boxes of `box_cols` by `box_rows`; what lies outside reads as zero and is not written.
int encode_map(CUtensorMap* tm, CUtensorMapDataType type, int es, const void* p, int64_t rows, int64_t cols, int64_t stride,
               int box_rows, int box_cols, CUtensorMapSwizzle swizzle) {
  EncodeTiledFn fn = get_encode_fn();
  if (!fn) { set_error("cuTensorMapEncodeTiled is not available from the driver"); return XDIT_E_DRIVER; }
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)(rows > 1 ? stride * es : (cols * es + 15) / 16 * 16)};  // a single row is never stepped
  cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows}, estr[2] = {1, 1};
  CUresult r = fn(tm, type, 2, const_cast<void*>(p), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("cuTensorMapEncodeTiled failed with CUresult %d (%lld x %lld, stride %lld)", (int)r, (long long)rows,
              (long long)cols, (long long)stride);
    return XDIT_E_DRIVER;
  }
  return XDIT_OK;
}

// The attribute is per device; set once per device, under a lock (calls may come from several threads).
template <auto Kernel>
int configure_smem(int bytes) {
  static std::mutex mu;
  static bool configured[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
  std::lock_guard<std::mutex> lk(mu);
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return cuda_fail(e, "fp8 linear smem attribute");
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  return XDIT_OK;
}

// CTAs that share the K axis of a tile when there are `tiles` of them: split in two up to three CTAs for two SMs, in four
// up to one for each, in eight up to three quarters of that, while a CTA keeps four steps.  Two CTAs fit an SM, but a
// cluster takes its places in one group of SMs, and what does not fit starts when others have ended (2 rows of 5120 to 4608:
// 36 tiles by 8 13.3 us, by 4 9.5; 2 rows to 9216: 72 by 4 16.8, by 2 12.8; 64 rows to 2304: 18 by 8 15.8, by 4 11.8; 2 rows
// of 13,824 to 1536: 12 by 8 9.8, by 4 12.1; 320 rows of 5120 to 2304: 90 by 2 20.2, whole 23.9).
int rows_splits(int64_t tiles, int kb, int sms) {
  int splits = 1;
  while (splits < kMaxSplits && tiles * splits * 2 <= (splits == 1 ? sms + sms / 2 : splits == 2 ? sms : sms * 3 / 4) && kb / (splits * 2) >= 4) splits *= 2;
  return splits;
}

// Few rows, or few tiles: NB the smallest of 16, 32, 64 that holds the rows, tiles of 64 above.
template <int NB>
int launch_rows(GemmArgs& a, const xdit_fp8_linear_params& p, int sms, bool after_quantise, cudaStream_t stream) {
  using L = RowsLayout<NB>;
  const CUtensorMapDataType u8 = CU_TENSOR_MAP_DATA_TYPE_UINT8;
  int rc;
  if ((rc = encode_map(&a.tm_x, u8, 1, p.x, p.M, p.K, p.x_stride_row, NB, kBK, CU_TENSOR_MAP_SWIZZLE_128B))) return rc;
  if ((rc = encode_map(&a.tm_w, u8, 1, p.w, p.N, p.K, p.w_stride_row, 128, kBK, CU_TENSOR_MAP_SWIZZLE_128B))) return rc;
  const int nt = (p.N + 127) / 128, mt = (p.M + NB - 1) / NB;
  a.splits = rows_splits((int64_t)nt * mt, a.kb, sms);
  if ((rc = configure_smem<fp8_rows_kernel<NB>>(L::kSmem))) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(nt * a.splits), (unsigned)mt);
  cfg.blockDim = dim3(kRowsThreads);
  cfg.dynamicSmemBytes = L::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = a.splits;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = after_quantise ? 2 : 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, fp8_rows_kernel<NB>, a);
  if (e != cudaSuccess) return cuda_fail(e, "fp8_rows_kernel launch");
  return XDIT_OK;
}

}  // namespace
}  // namespace xdit

using namespace xdit;

extern "C" int xdit_fp8_linear(const struct xdit_fp8_linear_params* p, void* stream) {
  const char* who = "xdit_fp8_linear";
  if (!p) { set_error("%s: NULL params", who); return XDIT_E_NULL; }
  if (p->M < 0 || p->N < 1 || p->K < 16 || p->K % 16 || (p->out_q && p->N % 16)) {
    set_error("%s: M=%d N=%d K=%d (K a multiple of 16; N too where the result is e4m3 rows)", who, p->M, p->N, p->K);
    return XDIT_E_SHAPE;
  }
  if (p->activation != XDIT_ACT_NONE && p->activation != XDIT_ACT_GELU_TANH) { set_error("%s: unknown activation %d", who, p->activation); return XDIT_E_DTYPE; }
  const int es = p->out_q ? 1 : dtype_size(p->out_dtype);
  if (!es || (p->bias && !dtype_size(p->bias_dtype))) { set_error("%s: bad dtype of the result (%d) or bias (%d)", who, p->out_dtype, p->bias_dtype); return XDIT_E_DTYPE; }
  if (p->M == 0) return XDIT_OK;
  if (!p->x || !p->x_scale || !p->w || !p->w_scale || (!p->out && !p->out_q) || (p->out_q && !p->out_scale)) { set_error("%s: NULL pointer", who); return XDIT_E_NULL; }
  if ((((uintptr_t)p->x) & 15) || (((uintptr_t)p->w) & 15) || (p->M > 1 && (p->x_stride_row % 16 || p->x_stride_row < p->K)) ||
      (p->N > 1 && (p->w_stride_row % 16 || p->w_stride_row < p->K)) || (p->out_q && ((((uintptr_t)p->out_q) & 15) || p->out_scale_ld < p->M))) {
    set_error("%s: rows of x, w and out_q must start on 16-byte boundaries, out_scale_ld be at least M", who);
    return XDIT_E_ALIGN;
  }
  if ((((uintptr_t)p->x_scale | (uintptr_t)p->w_scale | (uintptr_t)p->out_scale) & 3) ||
      (p->bias && ((uintptr_t)p->bias & (dtype_size(p->bias_dtype) - 1)))) {
    set_error("%s: scales or bias are not aligned to their elements", who);
    return XDIT_E_ALIGN;
  }
  if (p->raw && (p->x_scale_stride_row != 1 || p->x_stride_row != p->K || p->raw_s < 0 || (p->raw_s && p->M % p->raw_s))) {
    set_error("%s: x is quantised into contiguous rows with scales stored block by block; raw_s=%d of M=%d", who, p->raw_s, p->M);
    return XDIT_E_SHAPE;
  }
  if (!p->out_q && (((uintptr_t)p->out) % es || (p->M > 1 && p->out_stride_row < p->N))) { set_error("%s: out pointer or row stride", who); return XDIT_E_ALIGN; }
  if (p->status_host) {
    const int32_t code = *reinterpret_cast<const volatile int32_t*>(p->status_host);
    if (code != 0) {
      set_error("%s: an earlier launch gave up a bounded wait (code %d); nothing is launched until the status words "
                "are cleared", who, code);
      return XDIT_E_KERNEL_TIMEOUT;
    }
  }
  const void* result = p->out_q ? p->out_q : p->out;
  if (result == p->x || result == p->w || (p->out_q && (p->out_scale == p->x_scale || p->out_scale == p->w_scale))) {
    set_error("%s: the result lies on x, w or their scales, which are read until the last tile is done", who);
    return XDIT_E_SHAPE;
  }
  int sms = 0;
  int rc = check_device(&sms);
  if (rc) return rc;
  const bool quantise = p->raw != nullptr;
  if (quantise) {
    rc = launch_quantize_rows(who, p->raw, p->raw_stride_b, p->raw_stride_row, p->raw_dtype, p->raw_s ? p->M / p->raw_s : 1,
                              p->raw_s ? p->raw_s : p->M, p->K, const_cast<void*>(p->x), const_cast<float*>(p->x_scale),
                              p->x_scale_stride_block, stream);
    if (rc) return rc;
  }
  GemmArgs a;
  memset(&a, 0, sizeof(a));
  a.M = p->M; a.N = p->N;
  a.kb = (p->K + kBK - 1) / kBK;
  a.mt = (p->M + kBM - 1) / kBM;
  a.nt = (p->N + kBN - 1) / kBN;
  a.xs = p->x_scale; a.xs_srow = p->x_scale_stride_row; a.xs_skb = p->x_scale_stride_block;
  a.ws = p->w_scale; a.ws_snb = p->w_scale_stride_row; a.ws_skb = p->w_scale_stride_block;
  a.bias = p->bias; a.bias_dtype = p->bias_dtype; a.act = p->activation; a.out_dtype = p->out_dtype;
  a.out = p->out; a.out_srow = p->out_stride_row;
  a.out_q = (uint8_t*)p->out_q; a.out_scale = p->out_scale; a.out_scale_ld = p->out_scale_ld;
  a.wide = ((uintptr_t)p->out) % 16 == 0 && (p->M == 1 || (p->out_stride_row * es) % 16 == 0);
  a.status = p->status; a.status_host = p->status_host;
  a.wait_limit_ns = p->wait_limit_ns ? p->wait_limit_ns : kWaitLimitNs;
  a.selftest_stall = p->selftest_stall;
  if (p->M <= 64) {
    if (p->M <= 16) return launch_rows<16>(a, *p, sms, quantise, (cudaStream_t)stream);
    if (p->M <= 32) return launch_rows<32>(a, *p, sms, quantise, (cudaStream_t)stream);
    return launch_rows<64>(a, *p, sms, quantise, (cudaStream_t)stream);
  }
  // Few tiles of a long K axis: here a tile's steps follow one another in one CTA (about 6.5 us + 0.42 us a step), there a
  // cluster shares them (8.5 us + 0.55 us a step of a CTA).  It is worth it from two CTAs a tile and 16 steps on (65 rows of
  // 4096 to 5120: 17.7 us split and 20.0 whole, of 13,824 38.5 and 56.0, 256 rows of 6528 to 352 11.8 and 27.1; below, 65
  // rows of 1152 to 1152 10.0 and 8.7).
  if (a.kb >= 16 && rows_splits((int64_t)((p->N + 127) / 128) * ((p->M + 63) / 64), a.kb, sms) > 1)
    return launch_rows<64>(a, *p, sms, quantise, (cudaStream_t)stream);
  // Pairs of CTAs take tiles of 256 rows, single CTAs of 128.  A pair reads W once for twice the rows, but starts and
  // ends later and wastes more of a last, partly filled wave: it is worth it from four waves on (5120 x 5120: 2048
  // rows 58 us by pairs and 56 by single CTAs, 4096 rows 98 and 103, 18,900 rows 409 and 437).
  const int mt2 = (p->M + 2 * kBM - 1) / (2 * kBM);
  const bool pairs = (int64_t)a.mt * a.nt > 3 * sms;
  if (pairs) a.mt = mt2;
  const int64_t band = kBandBytes / ((int64_t)p->K * (pairs ? 2 * kBM : kBM));
  a.band = (int)(band < 1 ? 1 : band > a.mt ? a.mt : band);
  const CUtensorMapDataType u8 = CU_TENSOR_MAP_DATA_TYPE_UINT8, u16 = CU_TENSOR_MAP_DATA_TYPE_UINT16;
  if ((rc = encode_map(&a.tm_x, u8, 1, p->x, p->M, p->K, p->x_stride_row, kBM, kBK, CU_TENSOR_MAP_SWIZZLE_128B))) return rc;
  if ((rc = encode_map(&a.tm_w, u8, 1, p->w, p->N, p->K, p->w_stride_row, pairs ? kBN / 2 : kBN, kBK, CU_TENSOR_MAP_SWIZZLE_128B))) return rc;
  a.tma_out = p->out_q || (a.wide && es == 2);
  if (p->out_q)
    rc = encode_map(&a.tm_out, u8, 1, p->out_q, p->M, p->N, p->N, 32, kCols, CU_TENSOR_MAP_SWIZZLE_128B);
  else if (a.tma_out)
    rc = encode_map(&a.tm_out, u16, 2, p->out, p->M, p->N, p->out_stride_row, 32, 64, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc) return rc;
  const int64_t tiles = (int64_t)a.mt * a.nt;
  if (tiles > 0x3fffffffll) { set_error("%s: too many tiles", who); return XDIT_E_SHAPE; }
  if ((rc = pairs ? configure_smem<fp8_gemm_kernel<true>>(GemmLayout<true>::kSmem)
                  : configure_smem<fp8_gemm_kernel<false>>(GemmLayout<false>::kSmem))) return rc;
  const int most = pairs ? sms / 2 : sms, size = pairs ? 2 : 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(size * (tiles < most ? tiles : most)));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = pairs ? GemmLayout<true>::kSmem : GemmLayout<false>::kSmem;
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = size;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = quantise ? 2 : 1;
  cudaError_t e = pairs ? cudaLaunchKernelEx(&cfg, fp8_gemm_kernel<true>, a) : cudaLaunchKernelEx(&cfg, fp8_gemm_kernel<false>, a);
  if (e != cudaSuccess) return cuda_fail(e, "fp8_gemm_kernel launch");
  return XDIT_OK;
}
