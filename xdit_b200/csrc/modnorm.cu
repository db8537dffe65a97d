// The steps of a DiT block between two sub-layers in one pass over a token's row:
//   h = residual_scale * residual + gate * post(branch)      post: none, LayerNorm or RMSNorm
//   z = norm(h) * (1 + scale) + shift                        norm: none, LayerNorm or RMSNorm
// with h and z written, or z as e4m3 rows with one scale for each block of 128 (fp8_quant.cuh) where
// an 8-bit projection follows.  gate, scale and shift hold one row for all tokens, for each sample, or
// for each token.
//
// HBM-bound: residual and branch are read once, h and z written once; the row stays in registers (fp32,
// unrounded) between the sums and the writes.  LayerNorm takes the mean first and then the squares of the
// centred values, both from registers, so a row with a large mean loses nothing to cancellation.
#include <cstring>

#include "fp8_quant.cuh"

namespace xdit {
namespace {

struct RowVec {  // a row of C values: the same for all, or with a stride for samples or tokens
  const void* ptr;
  int64_t stride_b, stride_row;
  int32_t f32;
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

// V consecutive values at element `at` of a row that is read once: 16-byte accesses that stay out of L1,
// which keeps its room for the modulation rows.
template <typename T, int V>
__device__ __forceinline__ void load_row(const T* p, int at, float (&x)[V]) {
  if constexpr (V == 1) {
    x[0] = Io<T>::get(p[at]);
  } else {
    constexpr int kWords = V * sizeof(T) / 16;
    uint4 w[kWords];
#pragma unroll
    for (int i = 0; i < kWords; ++i)
      asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(w[i].x), "=r"(w[i].y), "=r"(w[i].z), "=r"(w[i].w) : "l"(reinterpret_cast<const uint4*>(p + at) + i));
    const T* t = reinterpret_cast<const T*>(w);
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = Io<T>::get(t[i]);
  }
}
template <typename T, int V>
__device__ __forceinline__ void store_row(T* p, int at, const float (&x)[V]) {
  if constexpr (V == 1) {
    p[at] = Io<T>::put(x[0]);
  } else {
    constexpr int kWords = V * sizeof(T) / 16;
    uint4 w[kWords];
    T* t = reinterpret_cast<T*>(w);
#pragma unroll
    for (int i = 0; i < V; ++i) t[i] = Io<T>::put(x[i]);
#pragma unroll
    for (int i = 0; i < kWords; ++i) *(reinterpret_cast<uint4*>(p + at) + i) = w[i];
  }
}
template <typename T, int V>
__device__ __forceinline__ void load_plain(const T* p, int at, float (&x)[V]) {
  if constexpr (V == 1) {
    x[0] = Io<T>::get(__ldg(p + at));
  } else {
    constexpr int kWords = V * sizeof(T) / 16;
    uint4 w[kWords];
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = __ldg(reinterpret_cast<const uint4*>(p + at) + i);
    const T* t = reinterpret_cast<const T*>(w);
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = Io<T>::get(t[i]);
  }
}
template <typename T, int V>
__device__ __forceinline__ void load_vec(const RowVec& v, int64_t off, int at, float (&x)[V]) {
  if (v.f32) load_plain<float, V>(reinterpret_cast<const float*>(v.ptr) + off, at, x);
  else load_plain<T, V>(reinterpret_cast<const T*>(v.ptr) + off, at, x);
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

// Mean (LayerNorm; 0 for RMSNorm) and reciprocal root of the mean square of a row held in registers.
template <int V, int TPR, int VPT>
__device__ __forceinline__ void row_stats(const NormArgs& a, int how, const float (&x)[VPT][V], int t, float* red,
                                          int& turn, float& mean, float& rstd) {
  mean = 0.f;
  if (how == XDIT_NORM_LAYER) {
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < VPT; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) sum += x[k][i];  // vectors behind the row are zero
    mean = row_sum<TPR>(sum, red, turn) / (float)a.C;
  }
  float sq = 0.f;
#pragma unroll
  for (int k = 0; k < VPT; ++k)
    if (t + TPR * k < a.nvec) {
#pragma unroll
      for (int i = 0; i < V; ++i) sq = fmaf(x[k][i] - mean, x[k][i] - mean, sq);
    }
  rstd = rsqrtf(row_sum<TPR>(sq, red, turn) / (float)a.C + a.eps);
}

template <int TPR> constexpr int kRowsPerCta = TPR == 32 ? 4 : 1;

template <typename T, int V, int TPR, int VPT>
__global__ void __launch_bounds__(TPR * kRowsPerCta<TPR>)
gated_residual_norm_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float red[2 * (TPR / 32)];
  constexpr int kRows = kRowsPerCta<TPR>;
  const int t = threadIdx.x % TPR;
  int turn = 0;
  for (int64_t r = (int64_t)blockIdx.x * kRows + threadIdx.x / TPR; r < a.rows; r += (int64_t)gridDim.x * kRows) {
    const int b = (int)r / a.s, row = (int)r - b * a.s;
    auto at_vec = [&](const RowVec& v) { return b * v.stride_b + row * v.stride_row; };
    float h[VPT][V];
    const T* res = reinterpret_cast<const T*>(a.residual) + b * a.r_sb + row * a.r_srow;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const int idx = t + TPR * k;
#pragma unroll
      for (int i = 0; i < V; ++i) h[k][i] = 0.f;
      if (idx < a.nvec) load_row<T, V>(res, idx * V, h[k]);
    }
    if (a.branch) {
      float y[VPT][V];
      const T* br = reinterpret_cast<const T*>(a.branch) + b * a.y_sb + row * a.y_srow;
#pragma unroll
      for (int k = 0; k < VPT; ++k) {
        const int idx = t + TPR * k;
#pragma unroll
        for (int i = 0; i < V; ++i) y[k][i] = 0.f;
        if (idx < a.nvec) load_row<T, V>(br, idx * V, y[k]);
      }
      float mean = 0.f, rstd = 1.f;
      if (a.post != XDIT_NORM_NONE) row_stats<V, TPR, VPT>(a, a.post, y, t, red, turn, mean, rstd);
#pragma unroll
      for (int k = 0; k < VPT; ++k) {
        const int idx = t + TPR * k;
        if (idx >= a.nvec) continue;
        float v[V];
        if (a.post != XDIT_NORM_NONE) {
#pragma unroll
          for (int i = 0; i < V; ++i) y[k][i] = (y[k][i] - mean) * rstd;
          if (a.post_weight.ptr) {
            load_vec<T, V>(a.post_weight, 0, idx * V, v);
#pragma unroll
            for (int i = 0; i < V; ++i) y[k][i] *= v[i];
          }
          if (a.post_bias.ptr) {
            load_vec<T, V>(a.post_bias, 0, idx * V, v);
#pragma unroll
            for (int i = 0; i < V; ++i) y[k][i] += v[i];
          }
        }
        if (a.gate.ptr) {
          load_vec<T, V>(a.gate, at_vec(a.gate), idx * V, v);
#pragma unroll
          for (int i = 0; i < V; ++i) y[k][i] *= v[i];
        }
#pragma unroll
        for (int i = 0; i < V; ++i) h[k][i] = fmaf(a.residual_scale, h[k][i], y[k][i]);
      }
    }
    if (a.out_h) {
      T* o = reinterpret_cast<T*>(a.out_h) + b * a.h_sb + row * a.h_srow;
#pragma unroll
      for (int k = 0; k < VPT; ++k)
        if (t + TPR * k < a.nvec) store_row<T, V>(o, (t + TPR * k) * V, h[k]);
    }
    if (a.norm == XDIT_NORM_NONE) continue;
    float mean, rstd;
    row_stats<V, TPR, VPT>(a, a.norm, h, t, red, turn, mean, rstd);
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const int idx = t + TPR * k;
      if (idx < a.nvec) {
        float v[V];
#pragma unroll
        for (int i = 0; i < V; ++i) h[k][i] = (h[k][i] - mean) * rstd;
        if (a.weight.ptr) {
          load_vec<T, V>(a.weight, 0, idx * V, v);
#pragma unroll
          for (int i = 0; i < V; ++i) h[k][i] *= v[i];
        }
        if (a.bias.ptr) {
          load_vec<T, V>(a.bias, 0, idx * V, v);
#pragma unroll
          for (int i = 0; i < V; ++i) h[k][i] += v[i];
        }
        if (a.scale.ptr) {
          load_vec<T, V>(a.scale, at_vec(a.scale), idx * V, v);
#pragma unroll
          for (int i = 0; i < V; ++i) h[k][i] = fmaf(h[k][i], v[i], h[k][i]);
        }
        if (a.shift.ptr) {
          load_vec<T, V>(a.shift, at_vec(a.shift), idx * V, v);
#pragma unroll
          for (int i = 0; i < V; ++i) h[k][i] += v[i];
        }
        if (!a.out_q)
          store_row<T, V>(reinterpret_cast<T*>(a.out_z) + b * a.z_sb + row * a.z_srow, idx * V, h[k]);
      }
      if constexpr (V == 8) {
        if (a.out_q) {
          // 16 consecutive threads hold a block of 128; those behind the row add nothing to its maximum
          float top = 0.f;
          if (idx < a.nvec) {
#pragma unroll
            for (int i = 0; i < 8; ++i) top = amax_nan(top, h[k][i]);
          }
#pragma unroll
          for (int m = 8; m > 0; m >>= 1) top = amax_nan(top, __shfl_xor_sync(0xffffffffu, top, m));
          float inv;
          const float sc = block_scale(top, inv);
          if (idx < a.nvec) {
            uint2 q;
            q.x = pack_e4m3(h[k][0] * inv, h[k][1] * inv, h[k][2] * inv, h[k][3] * inv);
            q.y = pack_e4m3(h[k][4] * inv, h[k][5] * inv, h[k][6] * inv, h[k][7] * inv);
            *reinterpret_cast<uint2*>(a.out_q + r * a.C + idx * 8) = q;
            if (idx % 16 == 0) a.out_scale[(idx / 16) * a.scale_ld + r] = sc;
          }
        }
      }
    }
  }
}

// Rows of a tensor to e4m3 with one scale for each block of 128: 16 threads per block of 128.
template <typename T>
__global__ void __launch_bounds__(256)
quantize_rows_kernel(const T* x, int64_t sb, int64_t srow, int s, int64_t rows, int K, uint8_t* q, float* scale,
                     int64_t ld) {
  const int kb = (K + kBlock - 1) / kBlock;
  const int64_t items = rows * kb * 16;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < ((items + 31) / 32) * 32; i += (int64_t)gridDim.x * 256) {
    const int64_t blk = i >> 4, r = blk / kb;
    const int c = (int)(blk - r * kb), col = c * kBlock + (int)(i & 15) * 8;
    const bool live = i < items && col < K;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (live) load_row<T, 8>(x + (r / s) * sb + (r % s) * srow, col, v);
    float top = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = amax_nan(top, v[j]);
#pragma unroll
    for (int m = 8; m > 0; m >>= 1) top = amax_nan(top, __shfl_xor_sync(0xffffffffu, top, m));
    float inv;
    const float sc = block_scale(top, inv);
    if (live) {
      uint2 o;
      o.x = pack_e4m3(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
      o.y = pack_e4m3(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv);
      *reinterpret_cast<uint2*>(q + r * K + col) = o;
      if ((i & 15) == 0) scale[c * ld + r] = sc;
    }
  }
}

// A weight [N, K] to e4m3 with one scale for each block of 128 x 128: one CTA per block, which a thread
// crosses in pieces of 8 columns.
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
    if (row0 + 16 * k < N && col < K) load_row<T, 8>(w + (row0 + 16 * k) * srow, col, v[k]);
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

template <typename T, int V, int TPR, int VPT>
cudaError_t launch(const NormArgs& a, int sms, cudaStream_t stream) {
  constexpr int kRows = kRowsPerCta<TPR>, kThreads = TPR * kRows;
  int64_t ctas = ((int64_t)a.rows + kRows - 1) / kRows, most = (int64_t)sms * (2048 / kThreads);
  gated_residual_norm_kernel<T, V, TPR, VPT><<<(int)(ctas < most ? ctas : most), kThreads, 0, stream>>>(a);
  return cudaGetLastError();
}

// Threads and vectors per thread of a row: as few threads as hold it in five vectors each (one warp up to
// 1280 values: no barrier between a row's loads and its stores).
template <typename T>
cudaError_t dispatch(const NormArgs& a, int V, int sms, cudaStream_t stream) {
#define XDIT_VPT5(V, TPR)                                       \
  switch ((a.nvec + TPR - 1) / TPR) {                           \
    case 1: return launch<T, V, TPR, 1>(a, sms, stream);        \
    case 2: return launch<T, V, TPR, 2>(a, sms, stream);        \
    case 3: return launch<T, V, TPR, 3>(a, sms, stream);        \
    case 4: return launch<T, V, TPR, 4>(a, sms, stream);        \
    default: return launch<T, V, TPR, 5>(a, sms, stream);       \
  }
  if (V == 8) {
    if (a.nvec <= 160) XDIT_VPT5(8, 32)
    if (a.nvec <= 640) XDIT_VPT5(8, 128)
    XDIT_VPT5(8, 512)
  }
#undef XDIT_VPT5
  if (a.nvec <= 1024) return launch<T, 1, 128, 8>(a, sms, stream);
  if (a.nvec <= 4096) return launch<T, 1, 512, 8>(a, sms, stream);
  return launch<T, 1, 512, 40>(a, sms, stream);
}

bool aligned_rows(const void* p, int64_t sb, int64_t srow, int es, const xdit_norm_params& q) {
  return ((uintptr_t)p & 15) == 0 && (q.B == 1 || (sb * es) % 16 == 0) && (q.s == 1 || (srow * es) % 16 == 0);
}

}  // namespace

int launch_norm(const xdit_norm_params& p, cudaStream_t stream) {
  const char* who = "xdit_gated_residual_norm";
  const int es = dtype_size(p.dtype);
  if (!es) { set_error("%s: bad dtype %d", who, p.dtype); return XDIT_E_DTYPE; }
  if (p.B < 0 || p.s < 0 || p.C < 1 || p.C > XDIT_NORM_MAX_C || (int64_t)p.B * p.s > 0x7fffffffll) {
    set_error("%s: B=%d s=%d C=%d (C at most %d)", who, p.B, p.s, p.C, XDIT_NORM_MAX_C);
    return XDIT_E_SHAPE;
  }
  if (p.norm < XDIT_NORM_NONE || p.norm > XDIT_NORM_RMS || p.post_norm < XDIT_NORM_NONE || p.post_norm > XDIT_NORM_RMS) {
    set_error("%s: unknown norm %d or post_norm %d", who, p.norm, p.post_norm);
    return XDIT_E_DTYPE;
  }
  if (p.norm == XDIT_NORM_NONE && !p.branch) { set_error("%s: nothing to do without a norm and a branch", who); return XDIT_E_SHAPE; }
  if (p.B == 0 || p.s == 0) return XDIT_OK;
  if (!p.residual || (p.branch && !p.out_residual) || (p.norm != XDIT_NORM_NONE && !p.out && !p.out_q) ||
      (p.out_q && !p.out_scale)) {
    set_error("%s: NULL residual or output", who);
    return XDIT_E_NULL;
  }
  NormArgs a;
  memset(&a, 0, sizeof(a));
  bool wide = p.C % 8 == 0;
  wide &= aligned_rows(p.residual, p.residual_stride_b, p.residual_stride_row, es, p);
  if (p.branch) wide &= aligned_rows(p.branch, p.branch_stride_b, p.branch_stride_row, es, p);
  if (p.out_residual) wide &= aligned_rows(p.out_residual, p.out_residual_stride_b, p.out_residual_stride_row, es, p);
  if (p.out && !p.out_q) wide &= aligned_rows(p.out, p.out_stride_b, p.out_stride_row, es, p);
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
    to[i]->f32 = in[i]->dtype == XDIT_F32;
    wide &= aligned_rows(in[i]->ptr, in[i]->stride_b, in[i]->stride_row, dtype_size(in[i]->dtype), p);
  }
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
  a.nvec = wide ? p.C / 8 : p.C;
  a.post = p.post_norm; a.norm = p.norm;
  a.residual_scale = p.residual_scale; a.eps = p.eps;
  cudaError_t e = p.dtype == XDIT_BF16  ? dispatch<__nv_bfloat16>(a, wide ? 8 : 1, sms, stream)
                  : p.dtype == XDIT_F16 ? dispatch<__half>(a, wide ? 8 : 1, sms, stream)
                                        : dispatch<float>(a, wide ? 8 : 1, sms, stream);
  if (e != cudaSuccess) return cuda_fail(e, "gated_residual_norm_kernel launch");
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
  const char* who = "xdit_quantize_rows";
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
  int sms = 0;
  int rc = check_device(&sms);
  if (rc) return rc;
  const int64_t blocks = (rows * ((K + kBlock - 1) / kBlock) * 16 + 255) / 256, most = (int64_t)sms * 32;
  const int grid = (int)(blocks < most ? blocks : most);
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == XDIT_BF16)
    quantize_rows_kernel<<<grid, 256, 0, st>>>((const __nv_bfloat16*)x, stride_b, stride_row, s, rows, K, (uint8_t*)q, scale, scale_ld);
  else if (dtype == XDIT_F16)
    quantize_rows_kernel<<<grid, 256, 0, st>>>((const __half*)x, stride_b, stride_row, s, rows, K, (uint8_t*)q, scale, scale_ld);
  else
    quantize_rows_kernel<<<grid, 256, 0, st>>>((const float*)x, stride_b, stride_row, s, rows, K, (uint8_t*)q, scale, scale_ld);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "quantize_rows_kernel launch");
  return XDIT_OK;
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
