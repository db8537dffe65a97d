// The steps of a DiT block between two sub-layers in one pass over a token's row:
//   h = residual_scale * residual + gate * post(branch)      post: none, LayerNorm or RMSNorm
//   z = norm(h) * (1 + scale) + shift                        norm: LayerNorm or RMSNorm (none: no z)
// with h and z written, or z as e4m3 rows with one scale for each block of 128 (fp8_quant.cuh) where
// an 8-bit projection follows.  gate, scale and shift hold one row for all tokens, for each sample, or
// for each token.
//
// HBM-bound: residual and branch are read once, h and z written once; the row stays in registers (fp32,
// unrounded) between the sums and the writes.  LayerNorm takes the mean first and then the squares of the
// centred values, both from registers, so a row with a large mean loses nothing to cancellation.
// 75,600 rows of 5120 in bf16 with modulation in fp32 (3.10 GB) take 500-551 us from box to box (5.6-6.2 TB/s, 0.86-0.94 of a
// copy).  A row takes registers, so an SM holds 16 warps (12 where a warp holds a row of 1152), and the row that each has on
// its way is what hides the latency (without it 760 us).  CTAs of 128 threads, four on an SM: three 633, five 616 (spills), six 731; three of 256 threads 600.  The
// modulation's 60 KB a row come from L1, more bytes than the row's own 40 KB: 551 us while they came 16 bytes a load,
// 610-637 with the row ahead in shared memory (five or six CTAs on an SM), which takes L1's room.
#include <cstring>

#include "fp8_quant.cuh"

namespace xdit {
namespace {

constexpr int kQuantThreads = 160;

struct RowVec {  // a row of C values: the same for all, or with a stride for samples or tokens
  const void* ptr;
  int64_t stride_b, stride_row;
  int32_t f32;  // 0: in the tensors' dtype, 1: fp32, 2: fp32 and every vector on a 32-byte boundary
};

struct NormArgs {
  const void *residual, *branch;
  int64_t r_sb, r_srow, y_sb, y_srow;
  void *out_h, *out_z;
  int64_t h_sb, h_srow, z_sb, z_srow;
  uint8_t* out_q;      // e4m3 [rows, C]
  float* out_scale;    // [C / 128 rounded up][scale_ld]
  int64_t scale_ld;
  RowVec post_weight, post_bias, gate, weight, bias, scale, shift;
  int32_t rows, s, C, nvec;
  int32_t post, norm;
  float residual_scale, eps;
};

template <typename T> struct Io;
template <> struct Io<float> {
  static __device__ __forceinline__ float get(float x) { return x; }
  static __device__ __forceinline__ float put(float x) { return x; }
};
template <> struct Io<__nv_bfloat16> {
  static __device__ __forceinline__ float get(__nv_bfloat16 x) { return __bfloat162float(x); }
  static __device__ __forceinline__ __nv_bfloat16 put(float x) { return __float2bfloat16_rn(x); }
};
template <> struct Io<__half> {
  static __device__ __forceinline__ float get(__half x) { return __half2float(x); }
  static __device__ __forceinline__ __half put(float x) { return __float2half_rn(x); }
};

// Two 16-bit values in a word <-> fp32 (taken as words: 16-bit values one by one cost twice the instructions).
template <typename T> struct Word;
template <> struct Word<__nv_bfloat16> {
  static __device__ __forceinline__ void get(uint32_t w, float& lo, float& hi) {
    lo = __uint_as_float(w << 16);
    hi = __uint_as_float(w & 0xffff0000u);
  }
  static __device__ __forceinline__ uint32_t put(float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  }
};
template <> struct Word<__half> {
  static __device__ __forceinline__ void get(uint32_t w, float& lo, float& hi) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    lo = f.x;
    hi = f.y;
  }
  static __device__ __forceinline__ uint32_t put(float lo, float hi) {
    __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  }
};

// The arithmetic runs on packed pairs, or on single values (V = 1).
template <int V> struct Lane { using E = uint64_t; static constexpr int N = V / 2; };
template <> struct Lane<1> { using E = float; static constexpr int N = 1; };
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void split(uint64_t x, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(x)); }
__device__ __forceinline__ uint64_t add(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mad(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ float add(float a, float b) { return a + b; }
__device__ __forceinline__ float mul(float a, float b) { return a * b; }
__device__ __forceinline__ float mad(float a, float b, float c) { return fmaf(a, b, c); }
template <typename E> __device__ __forceinline__ E both(float x);
template <> __device__ __forceinline__ uint64_t both<uint64_t>(float x) { return pair(x, x); }
template <> __device__ __forceinline__ float both<float>(float x) { return x; }
__device__ __forceinline__ float total(uint64_t x) {
  float lo, hi;
  split(x, lo, hi);
  return lo + hi;
}
__device__ __forceinline__ float total(float x) { return x; }

// V consecutive values as they lie in memory: V = 8 in 16-byte words, V = 2 in one access, V = 1 alone.
template <int BYTES> struct Pair { using type = uint32_t; };
template <> struct Pair<4> { using type = float2; };
template <typename T, int V> struct Raw {
  static constexpr int kWords = V * sizeof(T) / 16;
  uint4 w[kWords];
  // of a row that is read once: past L1, which keeps its room for the modulation rows
  __device__ __forceinline__ void load_once(const T* p) {
#pragma unroll
    for (int i = 0; i < kWords; ++i)
      asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(w[i].x), "=r"(w[i].y), "=r"(w[i].z), "=r"(w[i].w) : "l"(reinterpret_cast<const uint4*>(p) + i));
  }
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
  }
  // 32 bytes of a modulation row from a 32-byte boundary, in one load (two loads of 16 bytes lie 32 apart from thread to
  // thread and pass L1 at half the rate)
  __device__ __forceinline__ void load_wide(const T* p) {
    static_assert(kWords == 2);
    asm("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
        : "=r"(w[0].x), "=r"(w[0].y), "=r"(w[0].z), "=r"(w[0].w), "=r"(w[1].x), "=r"(w[1].y), "=r"(w[1].z), "=r"(w[1].w)
        : "l"(p));
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < kWords; ++i) *(reinterpret_cast<uint4*>(p) + i) = w[i];
  }
  __device__ __forceinline__ void get(uint64_t (&x)[V / 2]) const {
    const uint32_t* u = reinterpret_cast<const uint32_t*>(w);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      float lo, hi;
      if constexpr (sizeof(T) == 4) { lo = __uint_as_float(u[2 * i]); hi = __uint_as_float(u[2 * i + 1]); }
      else Word<T>::get(u[i], lo, hi);
      x[i] = pair(lo, hi);
    }
  }
  __device__ __forceinline__ void put(const uint64_t (&x)[V / 2]) {
    uint32_t* u = reinterpret_cast<uint32_t*>(w);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      float lo, hi;
      split(x[i], lo, hi);
      if constexpr (sizeof(T) == 4) { u[2 * i] = __float_as_uint(lo); u[2 * i + 1] = __float_as_uint(hi); }
      else u[i] = Word<T>::put(lo, hi);
    }
  }
};
template <typename T> struct Raw<T, 2> {  // two values in one word (16 bits each) or two
  using W = typename Pair<sizeof(T)>::type;
  W w;
  __device__ __forceinline__ void load_once(const T* p) { w = *reinterpret_cast<const W*>(p); }
  __device__ __forceinline__ void load(const T* p) { w = __ldg(reinterpret_cast<const W*>(p)); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<W*>(p) = w; }
  __device__ __forceinline__ void get(uint64_t (&x)[1]) const {
    float lo, hi;
    if constexpr (sizeof(T) == 4) { lo = w.x; hi = w.y; }
    else Word<T>::get(w, lo, hi);
    x[0] = pair(lo, hi);
  }
  __device__ __forceinline__ void put(const uint64_t (&x)[1]) {
    float lo, hi;
    split(x[0], lo, hi);
    if constexpr (sizeof(T) == 4) w = make_float2(lo, hi);
    else w = Word<T>::put(lo, hi);
  }
};
template <typename T> struct Raw<T, 1> {
  T w;
  __device__ __forceinline__ void load_once(const T* p) { w = *p; }
  __device__ __forceinline__ void load(const T* p) { w = __ldg(p); }
  __device__ __forceinline__ void store(T* p) const { *p = w; }
  __device__ __forceinline__ void get(float (&x)[1]) const { x[0] = Io<T>::get(w); }
  __device__ __forceinline__ void put(const float (&x)[1]) { w = Io<T>::put(x[0]); }
};

enum { kAdd, kMul, kScale };
// x (op) the modulation row `v`, which starts at element `at` for this thread: x + v, x v, x (1 + v).
template <int OP, typename R, bool WIDE, int V, int TPR, int VPT, typename E>
__device__ __forceinline__ void apply_as(const void* ptr, int64_t at, int t, int nvec, E (&x)[VPT][Lane<V>::N]) {
  const R* p = reinterpret_cast<const R*>(ptr) + at;
#pragma unroll
  for (int k = 0; k < VPT; ++k) {
    if (t + TPR * k >= nvec) continue;
    Raw<R, V> raw;
    if constexpr (WIDE) raw.load_wide(p + TPR * k * V);
    else raw.load(p + TPR * k * V);
    E v[Lane<V>::N];
    raw.get(v);
#pragma unroll
    for (int i = 0; i < Lane<V>::N; ++i)
      x[k][i] = OP == kAdd ? add(x[k][i], v[i]) : OP == kMul ? mul(x[k][i], v[i]) : mad(x[k][i], v[i], x[k][i]);
  }
}
template <int OP, typename T, int V, int TPR, int VPT, typename E>
__device__ __forceinline__ void apply(const RowVec& v, int b, int row, int t, int nvec, E (&x)[VPT][Lane<V>::N]) {
  if (!v.ptr) return;
  const int64_t at = b * v.stride_b + row * v.stride_row + t * V;
  if (v.f32 == 2) {
    if constexpr (V == 8) apply_as<OP, float, true, V, TPR, VPT>(v.ptr, at, t, nvec, x);
  } else if (v.f32) {
    apply_as<OP, float, false, V, TPR, VPT>(v.ptr, at, t, nvec, x);
  } else {
    apply_as<OP, T, false, V, TPR, VPT>(v.ptr, at, t, nvec, x);
  }
}

// Sum over the TPR threads of a row.  The shared buffer alternates, so one barrier per sum is enough: a
// buffer is written again only after the barrier of the sum in between.
template <int TPR>
__device__ __forceinline__ float row_sum(float x, float* red, int& turn) {
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) x += __shfl_xor_sync(0xffffffffu, x, m);
  if constexpr (TPR > 32) {
    float* buf = red + (turn & 1) * (TPR / 32);
    ++turn;
    if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = x;
    __syncthreads();
    x = buf[0];
#pragma unroll
    for (int i = 1; i < TPR / 32; ++i) x += buf[i];
  }
  return x;
}

// x <- (x - mean) / rms of a row held in registers (RMSNorm: the mean counts as 0).
template <int V, int TPR, int VPT, typename E>
__device__ __forceinline__ void normalise(const NormArgs& a, int how, E (&x)[VPT][Lane<V>::N], int t, float* red, int& turn) {
  if (how == XDIT_NORM_LAYER) {
    E sum = both<E>(0.f);
#pragma unroll
    for (int k = 0; k < VPT; ++k)
#pragma unroll
      for (int i = 0; i < Lane<V>::N; ++i) sum = add(sum, x[k][i]);  // vectors behind the row are zero
    const E mean = both<E>(-row_sum<TPR>(total(sum), red, turn) / (float)a.C);
#pragma unroll
    for (int k = 0; k < VPT; ++k)
#pragma unroll
      for (int i = 0; i < Lane<V>::N; ++i) x[k][i] = add(x[k][i], mean);
  }
  E sq = both<E>(0.f);
#pragma unroll
  for (int k = 0; k < VPT; ++k)
    if (t + TPR * k < a.nvec) {
#pragma unroll
      for (int i = 0; i < Lane<V>::N; ++i) sq = mad(x[k][i], x[k][i], sq);
    }
  const E rstd = both<E>(rsqrtf(row_sum<TPR>(total(sq), red, turn) / (float)a.C + a.eps));
#pragma unroll
  for (int k = 0; k < VPT; ++k)
#pragma unroll
    for (int i = 0; i < Lane<V>::N; ++i) x[k][i] = mul(x[k][i], rstd);
}

template <int TPR> constexpr int kRowsPerCta = TPR == 32 ? 4 : 1;

// A row's vectors are requested while the row before it is worked on.  Four CTAs on an SM for five vectors in 128 threads are
// the 16-bit types' best; fp32 rows of 4097-5120 values spill 192 bytes a thread there (75,600 of 5120 1576 us, 3.9 TB/s; of 4096
// values, without a spill, 5.4).
template <typename T, int V, int TPR, int VPT>
__global__ void __launch_bounds__(TPR * kRowsPerCta<TPR>, TPR == 128 && VPT == 5 ? 4 : 1)
gated_residual_norm_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float red[2 * (TPR / 32)];
  using E = typename Lane<V>::E;
  constexpr int N = Lane<V>::N, kRows = kRowsPerCta<TPR>;
  const int t = threadIdx.x % TPR;
  const int step = gridDim.x * kRows;
  int turn = 0;
  Raw<T, V> res[VPT], br[VPT];
  auto fetch = [&](int r) {
    const int b = r / a.s, row = r - b * a.s;
    const T* p = reinterpret_cast<const T*>(a.residual) + b * a.r_sb + row * a.r_srow + t * V;
#pragma unroll
    for (int k = 0; k < VPT; ++k)
      if (t + TPR * k < a.nvec) res[k].load_once(p + TPR * k * V);
    if (a.branch) {
      const T* q = reinterpret_cast<const T*>(a.branch) + b * a.y_sb + row * a.y_srow + t * V;
#pragma unroll
      for (int k = 0; k < VPT; ++k)
        if (t + TPR * k < a.nvec) br[k].load_once(q + TPR * k * V);
    }
  };
  auto write = [&](void* out, int64_t at, const E (&x)[VPT][N]) {
    T* o = reinterpret_cast<T*>(out) + at + t * V;
#pragma unroll
    for (int k = 0; k < VPT; ++k)
      if (t + TPR * k < a.nvec) {
        Raw<T, V> w;
        w.put(x[k]);
        w.store(o + TPR * k * V);
      }
  };
  int r = blockIdx.x * kRows + threadIdx.x / TPR;
  if (r < a.rows) fetch(r);
  for (; r < a.rows; r += step) {
    const int b = r / a.s, row = r - b * a.s;
    E h[VPT][N];
    auto zero = [&](E (&x)[VPT][N]) {
#pragma unroll
      for (int k = 0; k < VPT; ++k)
#pragma unroll
        for (int i = 0; i < N; ++i) x[k][i] = both<E>(0.f);
    };
    zero(h);
    if (a.branch) {
#pragma unroll
      for (int k = 0; k < VPT; ++k)
        if (t + TPR * k < a.nvec) br[k].get(h[k]);
      if (a.post != XDIT_NORM_NONE) {
        normalise<V, TPR, VPT>(a, a.post, h, t, red, turn);
        apply<kMul, T, V, TPR, VPT>(a.post_weight, b, row, t, a.nvec, h);
        apply<kAdd, T, V, TPR, VPT>(a.post_bias, b, row, t, a.nvec, h);
      }
      apply<kMul, T, V, TPR, VPT>(a.gate, b, row, t, a.nvec, h);
      const E rs = both<E>(a.residual_scale);
#pragma unroll
      for (int k = 0; k < VPT; ++k) {
        if (t + TPR * k >= a.nvec) {  // a normalised row has values behind its end
#pragma unroll
          for (int i = 0; i < N; ++i) h[k][i] = both<E>(0.f);
          continue;
        }
        E x[N];
        res[k].get(x);
#pragma unroll
        for (int i = 0; i < N; ++i) h[k][i] = mad(rs, x[i], h[k][i]);
      }
    } else {
#pragma unroll
      for (int k = 0; k < VPT; ++k)
        if (t + TPR * k < a.nvec) res[k].get(h[k]);
    }
    if (r + step < a.rows) fetch(r + step);
    if (a.out_h) write(a.out_h, b * a.h_sb + row * a.h_srow, h);
    if (a.norm == XDIT_NORM_NONE) continue;
    normalise<V, TPR, VPT>(a, a.norm, h, t, red, turn);
    apply<kMul, T, V, TPR, VPT>(a.weight, b, row, t, a.nvec, h);
    apply<kAdd, T, V, TPR, VPT>(a.bias, b, row, t, a.nvec, h);
    apply<kScale, T, V, TPR, VPT>(a.scale, b, row, t, a.nvec, h);
    apply<kAdd, T, V, TPR, VPT>(a.shift, b, row, t, a.nvec, h);
    if constexpr (V == 8) {
      if (a.out_q) {
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
          // 16 consecutive threads hold a block of 128; those behind the row add nothing to its maximum
          const int idx = t + TPR * k;
          float x[8], top = 0.f;
#pragma unroll
          for (int i = 0; i < 4; ++i) split(h[k][i], x[2 * i], x[2 * i + 1]);
          if (idx < a.nvec) {
#pragma unroll
            for (int i = 0; i < 8; i += 2) top = amax_nan(top, x[i], x[i + 1]);
          }
#pragma unroll
          for (int m = 8; m > 0; m >>= 1) top = amax_nan(top, __shfl_xor_sync(0xffffffffu, top, m));
          float inv;
          const float sc = block_scale(top, inv);
          if (idx < a.nvec) {
#pragma unroll
            for (int i = 0; i < 4; ++i) split(mul(h[k][i], both<E>(inv)), x[2 * i], x[2 * i + 1]);
            uint2 q;
            q.x = pack_e4m3(x[0], x[1], x[2], x[3]);
            q.y = pack_e4m3(x[4], x[5], x[6], x[7]);
            *reinterpret_cast<uint2*>(a.out_q + (int64_t)r * a.C + idx * 8) = q;
            if (idx % 16 == 0) a.out_scale[(idx / 16) * a.scale_ld + r] = sc;
          }
        }
        continue;
      }
    }
    write(a.out_z, b * a.z_sb + row * a.z_srow, h);
  }
}

// Rows of a tensor to e4m3 with one scale for each block of 128: a CTA walks whole rows, 16 threads hold a block, and
// four vectors of a thread are on their way at a time (HBM-bound: 75,600 x 5120 bf16, 1.16 GB, 192 us or 6.05 TB/s; one
// vector at a time 280 us).
template <typename T>
__global__ void __launch_bounds__(kQuantThreads)
quantize_rows_kernel(const T* x, int64_t sb, int64_t srow, int s, int64_t rows, int K, uint8_t* q, float* scale,
                     int64_t ld) {
  // a product that takes these rows may be launched now: it waits for this kernel's end before it reads them
  asm volatile("griddepcontrol.launch_dependents;");
  constexpr int kUnroll = 4;
  const int nvec = K / 8, t = threadIdx.x;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* src = x + (r / s) * sb + (r % s) * srow;
    for (int v0 = 0; v0 < nvec; v0 += kUnroll * kQuantThreads) {
      Raw<T, 8> w[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (v0 + u * kQuantThreads + t < nvec) w[u].load_once(src + (v0 + u * kQuantThreads + t) * 8);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int idx = v0 + u * kQuantThreads + t;
        if (v0 + u * kQuantThreads >= nvec) break;
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, top = 0.f;
        if (idx < nvec) {
          uint64_t p[4];
          w[u].get(p);
#pragma unroll
          for (int j = 0; j < 4; ++j) split(p[j], v[2 * j], v[2 * j + 1]);
        }
#pragma unroll
        for (int j = 0; j < 8; j += 2) top = amax_nan(top, v[j], v[j + 1]);
#pragma unroll
        for (int m = 8; m > 0; m >>= 1) top = amax_nan(top, __shfl_xor_sync(0xffffffffu, top, m));
        float inv;
        const float sc = block_scale(top, inv);
        if (idx < nvec) {
          uint2 o;
          o.x = pack_e4m3(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
          o.y = pack_e4m3(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv);
          *reinterpret_cast<uint2*>(q + r * K + idx * 8) = o;
          if ((idx & 15) == 0) scale[(idx >> 4) * ld + r] = sc;
        }
      }
    }
  }
}

// A weight [N, K] to e4m3 with one scale for each block of 128 x 128: one CTA per block, which a thread
// crosses in pieces of 8 columns (run once for a weight, so left simple).
template <typename T>
__global__ void __launch_bounds__(256)
quantize_weight_kernel(const T* w, int64_t srow, int N, int K, uint8_t* q, float* scale) {
  __shared__ float red[8];
  const int kb = (K + kBlock - 1) / kBlock;
  const int nb = blockIdx.x / kb, c = blockIdx.x - nb * kb;
  const int col = c * kBlock + (threadIdx.x & 15) * 8, row0 = nb * kBlock + (threadIdx.x >> 4);
  float v[8][8];
  float top = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[k][j] = 0.f;
    if (row0 + 16 * k < N && col < K) {
      Raw<T, 8> raw;
      uint64_t p[4];
      raw.load_once(w + (row0 + 16 * k) * srow + col);
      raw.get(p);
#pragma unroll
      for (int j = 0; j < 4; ++j) split(p[j], v[k][2 * j], v[k][2 * j + 1]);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) top = amax_nan(top, v[k][j]);
  }
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) top = amax_nan(top, __shfl_xor_sync(0xffffffffu, top, m));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 8; ++k) top = amax_nan(top, red[k]);
  float inv;
  const float sc = block_scale(top, inv);
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const int row = row0 + 16 * k;
    if (row >= N || col >= K) continue;
    uint2 o;
    o.x = pack_e4m3(v[k][0] * inv, v[k][1] * inv, v[k][2] * inv, v[k][3] * inv);
    o.y = pack_e4m3(v[k][4] * inv, v[k][5] * inv, v[k][6] * inv, v[k][7] * inv);
    *reinterpret_cast<uint2*>(q + (int64_t)row * K + col) = o;
  }
  if (threadIdx.x == 0) scale[blockIdx.x] = sc;
}

// CTAs of a kernel that an SM holds.
template <typename F>
int resident_ctas(F* kernel, int threads) {
  int n = 0;
  return cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, 0) == cudaSuccess && n > 0 ? n : 1;
}

template <typename T, int V, int TPR, int VPT>
cudaError_t launch(const NormArgs& a, int sms, cudaStream_t stream) {
  constexpr int kRows = kRowsPerCta<TPR>, kThreads = TPR * kRows;
  const int64_t ctas = ((int64_t)a.rows + kRows - 1) / kRows;
  // as many CTAs as run at a time: each walks its rows with the next one's loads in flight
  static const int resident = resident_ctas(gated_residual_norm_kernel<T, V, TPR, VPT>, kThreads);
  const int64_t most = (int64_t)sms * resident;
  gated_residual_norm_kernel<T, V, TPR, VPT><<<(int)(ctas < most ? ctas : most), kThreads, 0, stream>>>(a);
  return cudaGetLastError();
}

// Threads and vectors per thread of a row: as few threads as hold it in five vectors each (one warp up to
// 1280 values: no barrier between a row's loads and its stores).  Rows that 16-byte words do not fit go by pairs of
// values or, of odd width, value by value (190,568 rows of 234: 471 us by values in CTAs of 128, 145 us by pairs in warps,
// 202 us of 235 by values), in threads enough for few registers: 6000 rows of 6002 take 137 us by 7 pairs a thread, 211 us by
// 16 with the last ones idle; 3063 of 1155 by values 15.6 us by 10 a thread and 17.9 by 12.
template <typename T>
cudaError_t dispatch(const NormArgs& a, int V, int sms, cudaStream_t stream) {
  if (V == 8) {
    if (a.nvec <= 32) return launch<T, 8, 32, 1>(a, sms, stream);
    if (a.nvec <= 64) return launch<T, 8, 32, 2>(a, sms, stream);
    if (a.nvec <= 96) return launch<T, 8, 32, 3>(a, sms, stream);
    if (a.nvec <= 128) return launch<T, 8, 32, 4>(a, sms, stream);
    if (a.nvec <= 160) return launch<T, 8, 32, 5>(a, sms, stream);
    if (a.nvec <= 256) return launch<T, 8, 128, 2>(a, sms, stream);
    if (a.nvec <= 384) return launch<T, 8, 128, 3>(a, sms, stream);
    if (a.nvec <= 512) return launch<T, 8, 128, 4>(a, sms, stream);
    if (a.nvec <= 640) return launch<T, 8, 128, 5>(a, sms, stream);
    if (a.nvec <= 1024) return launch<T, 8, 512, 2>(a, sms, stream);
    if (a.nvec <= 1536) return launch<T, 8, 512, 3>(a, sms, stream);
    return launch<T, 8, 512, 4>(a, sms, stream);  // up to XDIT_NORM_MAX_C values
  }
  if (V == 2) {
    if (a.nvec <= 64) return launch<T, 2, 32, 2>(a, sms, stream);
    if (a.nvec <= 160) return launch<T, 2, 32, 5>(a, sms, stream);
    if (a.nvec <= 384) return launch<T, 2, 32, 12>(a, sms, stream);
    if (a.nvec <= 640) return launch<T, 2, 128, 5>(a, sms, stream);
    if (a.nvec <= 1280) return launch<T, 2, 128, 10>(a, sms, stream);
    if (a.nvec <= 3584) return launch<T, 2, 512, 7>(a, sms, stream);
    return launch<T, 2, 512, 16>(a, sms, stream);
  }
  if (a.nvec <= 128) return launch<T, 1, 32, 4>(a, sms, stream);
  if (a.nvec <= 384) return launch<T, 1, 32, 12>(a, sms, stream);
  if (a.nvec <= 768) return launch<T, 1, 32, 24>(a, sms, stream);
  if (a.nvec <= 1280) return launch<T, 1, 128, 10>(a, sms, stream);
  if (a.nvec <= 2560) return launch<T, 1, 512, 5>(a, sms, stream);
  if (a.nvec <= 4096) return launch<T, 1, 512, 8>(a, sms, stream);
  return launch<T, 1, 512, 32>(a, sms, stream);
}

// Low bits of all that a row's vectors start from, in elements of `es` bytes: 0 in the bits that all have clear.
uint64_t low_bits(const void* p, int64_t sb, int64_t srow, int es, const xdit_norm_params& q) {
  uint64_t low = (uint64_t)(uintptr_t)p;
  if (q.B > 1) low |= (uint64_t)(sb * es);
  if (q.s > 1) low |= (uint64_t)(srow * es);
  return low;
}

}  // namespace

int launch_norm(const xdit_norm_params& p, cudaStream_t stream) {
  const char* who = "xdit_gated_residual_norm";
  const int es = dtype_size(p.dtype);
  if (!es) { set_error("%s: bad dtype %d", who, p.dtype); return XDIT_E_DTYPE; }
  if (p.B < 0 || p.s < 0 || p.C < 1 || p.C > XDIT_NORM_MAX_C || (int64_t)p.B * p.s > 0x7f000000ll) {
    set_error("%s: B=%d s=%d C=%d (C at most %d)", who, p.B, p.s, p.C, XDIT_NORM_MAX_C);
    return XDIT_E_SHAPE;
  }
  if (p.norm < XDIT_NORM_NONE || p.norm > XDIT_NORM_RMS || p.post_norm < XDIT_NORM_NONE || p.post_norm > XDIT_NORM_RMS) {
    set_error("%s: unknown norm %d or post_norm %d", who, p.norm, p.post_norm);
    return XDIT_E_DTYPE;
  }
  if (p.B == 0 || p.s == 0) return XDIT_OK;  // (an empty tensor has no address: NULL does not mean absent here)
  if (p.norm == XDIT_NORM_NONE && !p.branch) { set_error("%s: nothing to do without a norm and a branch", who); return XDIT_E_SHAPE; }
  const bool post_rows = p.post_weight.ptr || p.post_bias.ptr, rows = p.weight.ptr || p.bias.ptr || p.scale.ptr || p.shift.ptr;
  if (p.norm == XDIT_NORM_NONE && (p.out || p.out_q || rows)) {
    set_error("%s: without a norm there is no second result, and weight, bias, scale and shift have nothing to apply to", who);
    return XDIT_E_SHAPE;
  }
  if ((p.post_norm == XDIT_NORM_NONE && post_rows) || (!p.branch && (p.post_norm != XDIT_NORM_NONE || p.gate.ptr))) {
    set_error("%s: post_weight and post_bias need a post norm; that and a gate need a branch", who);
    return XDIT_E_SHAPE;
  }
  if (!p.residual || (p.branch && !p.out_residual) || (p.norm != XDIT_NORM_NONE && !p.out && !p.out_q) ||
      (p.out_q && !p.out_scale)) {
    set_error("%s: NULL residual or output", who);
    return XDIT_E_NULL;
  }
  NormArgs a;
  memset(&a, 0, sizeof(a));
  // V = 8 takes 16-byte words everywhere, V = 2 the size of two elements
  uint64_t low = 0, low_pair = 0;
  bool off = false;  // a pointer between elements
  auto look = [&](const void* ptr, int64_t sb, int64_t srow, int size) {
    const uint64_t l = low_bits(ptr, sb, srow, size, p);
    low |= l;
    low_pair |= l & (uint64_t)(2 * size - 1);
    off |= ((uintptr_t)ptr & (size - 1)) != 0;
  };
  look(p.residual, p.residual_stride_b, p.residual_stride_row, es);
  if (p.branch) look(p.branch, p.branch_stride_b, p.branch_stride_row, es);
  if (p.out_residual) look(p.out_residual, p.out_residual_stride_b, p.out_residual_stride_row, es);
  if (p.out && !p.out_q) look(p.out, p.out_stride_b, p.out_stride_row, es);
  const xdit_row_vec* in[7] = {&p.post_weight, &p.post_bias, &p.gate, &p.weight, &p.bias, &p.scale, &p.shift};
  RowVec* to[7] = {&a.post_weight, &a.post_bias, &a.gate, &a.weight, &a.bias, &a.scale, &a.shift};
  for (int i = 0; i < 7; ++i) {
    if (!in[i]->ptr) continue;
    if (in[i]->dtype != p.dtype && in[i]->dtype != XDIT_F32) {
      set_error("%s: a modulation row has dtype %d: the tensors' dtype or fp32", who, in[i]->dtype);
      return XDIT_E_DTYPE;
    }
    to[i]->ptr = in[i]->ptr;
    to[i]->stride_b = in[i]->stride_b;
    to[i]->stride_row = in[i]->stride_row;
    const bool apart = (low_bits(in[i]->ptr, in[i]->stride_b, in[i]->stride_row, 4, p) & 31) != 0;
    to[i]->f32 = in[i]->dtype != XDIT_F32 ? 0 : apart ? 1 : 2;
    look(in[i]->ptr, in[i]->stride_b, in[i]->stride_row, dtype_size(in[i]->dtype));
  }
  const bool h_one = p.out_residual && ((p.B > 1 && !p.out_residual_stride_b) || (p.s > 1 && !p.out_residual_stride_row));
  const bool z_one = p.out && !p.out_q && ((p.B > 1 && !p.out_stride_b) || (p.s > 1 && !p.out_stride_row));
  if (h_one || z_one || (p.norm != XDIT_NORM_NONE && p.out && p.out == p.out_residual)) {
    set_error("%s: an output holds several rows in one place, or both outputs are one", who);
    return XDIT_E_SHAPE;
  }
  // In place: element by element in residual or branch.  Rows are read while others are written, so an output at the
  // address of either with other strides, or on a row of modulation, would be read as it changes.
  bool torn = false;
  auto place = [&](const void* o, int64_t sb, int64_t srow) {
    if (!o) return;
    auto on = [&](const void* x, int64_t xb, int64_t xrow) {
      torn |= o == x && ((p.B > 1 && sb != xb) || (p.s > 1 && srow != xrow));
    };
    on(p.residual, p.residual_stride_b, p.residual_stride_row);
    on(p.branch, p.branch_stride_b, p.branch_stride_row);
    for (const xdit_row_vec* v : in) torn |= o == v->ptr;
  };
  place(p.out_residual, p.out_residual_stride_b, p.out_residual_stride_row);
  if (!p.out_q) place(p.out, p.out_stride_b, p.out_stride_row);
  if (torn) {
    set_error("%s: an output lies on residual or branch with other strides, or on a row of modulation", who);
    return XDIT_E_SHAPE;
  }
  if (off) { set_error("%s: a pointer is not aligned to its elements", who); return XDIT_E_ALIGN; }
  const bool wide = p.C % 8 == 0 && (low & 15) == 0;
  if (!wide)
    for (RowVec* v : to) v->f32 = v->f32 != 0;  // 32 bytes are the width of V = 8
  const int V = wide ? 8 : p.C % 2 == 0 && low_pair == 0 ? 2 : 1;
  if (p.out_q && (!wide || p.C % 16 || ((uintptr_t)p.out_q & 15) || p.out_scale_ld < (int64_t)p.B * p.s)) {
    set_error("%s: e4m3 rows need C %% 16 == 0, 16-byte aligned rows and out_scale_ld of at least B*s", who);
    return XDIT_E_ALIGN;
  }
  int sms = 0;
  int rc = check_device(&sms);
  if (rc) return rc;
  a.residual = p.residual; a.r_sb = p.residual_stride_b; a.r_srow = p.residual_stride_row;
  a.branch = p.branch; a.y_sb = p.branch_stride_b; a.y_srow = p.branch_stride_row;
  a.out_h = p.out_residual; a.h_sb = p.out_residual_stride_b; a.h_srow = p.out_residual_stride_row;
  a.out_z = p.out; a.z_sb = p.out_stride_b; a.z_srow = p.out_stride_row;
  a.out_q = (uint8_t*)p.out_q; a.out_scale = p.out_scale; a.scale_ld = p.out_scale_ld;
  a.rows = p.B * p.s; a.s = p.s; a.C = p.C;
  a.nvec = p.C / V;
  a.post = p.post_norm; a.norm = p.norm;
  a.residual_scale = p.residual_scale; a.eps = p.eps;
  cudaError_t e = p.dtype == XDIT_BF16  ? dispatch<__nv_bfloat16>(a, V, sms, stream)
                  : p.dtype == XDIT_F16 ? dispatch<__half>(a, V, sms, stream)
                                        : dispatch<float>(a, V, sms, stream);
  if (e != cudaSuccess) return cuda_fail(e, "gated_residual_norm_kernel launch");
  return XDIT_OK;
}

int launch_quantize_rows(const char* who, const void* x, int64_t stride_b, int64_t stride_row, int32_t dtype, int32_t B,
                         int32_t s, int32_t K, void* q, float* scale, int64_t scale_ld, void* stream) {
  const int es = dtype_size(dtype);
  if (!es) { set_error("%s: bad dtype %d", who, dtype); return XDIT_E_DTYPE; }
  const int64_t rows = (int64_t)B * s;
  if (B < 0 || s < 0 || K < 16 || K % 16 || scale_ld < rows) {
    set_error("%s: B=%d s=%d K=%d (a multiple of 16) scale_ld=%lld (at least B*s)", who, B, s, K, (long long)scale_ld);
    return XDIT_E_SHAPE;
  }
  if (rows == 0) return XDIT_OK;
  if (!x || !q || !scale) { set_error("%s: NULL pointer", who); return XDIT_E_NULL; }
  if (((uintptr_t)x & 15) || ((uintptr_t)q & 15) || (B > 1 && (stride_b * es) % 16) || (s > 1 && (stride_row * es) % 16)) {
    set_error("%s: rows must start on 16-byte boundaries", who);
    return XDIT_E_ALIGN;
  }
  if (x == q) { set_error("%s: the e4m3 rows lie on those that are read", who); return XDIT_E_SHAPE; }
  int rc = check_device(nullptr);
  if (rc) return rc;
  const int grid = (int)(rows < 0x7fffffffll ? rows : 0x7fffffffll);
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == XDIT_BF16)
    quantize_rows_kernel<<<grid, kQuantThreads, 0, st>>>((const __nv_bfloat16*)x, stride_b, stride_row, s, rows, K, (uint8_t*)q, scale, scale_ld);
  else if (dtype == XDIT_F16)
    quantize_rows_kernel<<<grid, kQuantThreads, 0, st>>>((const __half*)x, stride_b, stride_row, s, rows, K, (uint8_t*)q, scale, scale_ld);
  else
    quantize_rows_kernel<<<grid, kQuantThreads, 0, st>>>((const float*)x, stride_b, stride_row, s, rows, K, (uint8_t*)q, scale, scale_ld);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "quantize_rows_kernel launch");
  return XDIT_OK;
}


}  // namespace xdit

using namespace xdit;

extern "C" {

int xdit_gated_residual_norm(const struct xdit_norm_params* p, void* stream) {
  if (!p) { set_error("xdit_gated_residual_norm: NULL params"); return XDIT_E_NULL; }
  return launch_norm(*p, (cudaStream_t)stream);
}

int xdit_quantize_rows(const void* x, int64_t stride_b, int64_t stride_row, int32_t dtype, int32_t B, int32_t s,
                       int32_t K, void* q, float* scale, int64_t scale_ld, void* stream) {
  return launch_quantize_rows("xdit_quantize_rows", x, stride_b, stride_row, dtype, B, s, K, q, scale, scale_ld, stream);
}

int xdit_quantize_weight(const void* w, int64_t stride_row, int32_t dtype, int32_t N, int32_t K, void* q, float* scale,
                         void* stream) {
  const char* who = "xdit_quantize_weight";
  const int es = dtype_size(dtype);
  if (!es) { set_error("%s: bad dtype %d", who, dtype); return XDIT_E_DTYPE; }
  if (N < 1 || K < 16 || K % 16) { set_error("%s: N=%d K=%d (a multiple of 16)", who, N, K); return XDIT_E_SHAPE; }
  if (!w || !q || !scale) { set_error("%s: NULL pointer", who); return XDIT_E_NULL; }
  if (((uintptr_t)w & 15) || ((uintptr_t)q & 15) || (N > 1 && (stride_row * es) % 16)) {
    set_error("%s: rows must start on 16-byte boundaries", who);
    return XDIT_E_ALIGN;
  }
  const int64_t blocks = (int64_t)((N + kBlock - 1) / kBlock) * ((K + kBlock - 1) / kBlock);
  if (blocks > 0x7fffffffll) { set_error("%s: too many blocks", who); return XDIT_E_SHAPE; }
  if (w == q) { set_error("%s: the e4m3 weight lies on the one that is read", who); return XDIT_E_SHAPE; }
  int rc = check_device(nullptr);
  if (rc) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == XDIT_BF16)
    quantize_weight_kernel<<<(int)blocks, 256, 0, st>>>((const __nv_bfloat16*)w, stride_row, N, K, (uint8_t*)q, scale);
  else if (dtype == XDIT_F16)
    quantize_weight_kernel<<<(int)blocks, 256, 0, st>>>((const __half*)w, stride_row, N, K, (uint8_t*)q, scale);
  else
    quantize_weight_kernel<<<(int)blocks, 256, 0, st>>>((const float*)w, stride_row, N, K, (uint8_t*)q, scale);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "quantize_weight_kernel launch");
  return XDIT_OK;
}

}  // extern "C"
