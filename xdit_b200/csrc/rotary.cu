// Rotary positions with several axes (text index; time, height, width of a video): every rotated pair
// (a, b) of a head belongs to one axis and has a frequency f, and a token at position p of that axis turns
// it by the angle p f:  (a, b) -> (a cos - b sin, a sin + b cos).
//
// The angles come from the positions inside the kernel (ids per token, or a grid that the token index
// walks), so no cos/sin tables are read.  An angle is a product of a position that may be large and a
// frequency near one; in 32 bits it would be wrong by p 2^-24 radians (0.06 at position 1e6), so the
// product is taken in 64 bits and counted in turns (f / 2 pi), the whole turns are dropped, and only the
// fraction goes to 32 bits for sincospi.
//
// HBM-bound: q and k are read and written once.  A thread owns one vector of one token's head (its
// column does not change from head to head) and walks the heads of q and k, so the angles are computed
// once per thread and stay in registers.
#include <cstring>

#include "common.cuh"

namespace xdit {
namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 4;  // heads whose vectors a thread has in flight

struct RotaryArgs {
  const char* src[2];
  char* dst[2];
  int64_t ss_b[2], ss_h[2], ss_row[2];  // elements
  int64_t ds_b[2], ds_h[2], ds_row[2];
  int32_t heads[2];
  int64_t rows;      // B * s
  int32_t s, D, rot;
  int32_t slots;     // vectors of a head that threads own
  int32_t splits, per_split;  // heads (of q and k together) are split over `splits` threads
  // positions
  const void* pos;
  int64_t pos_sb, pos_srow, pos_saxis;
  int32_t pos_kind, axes;
  int64_t grid[XDIT_ROTARY_MAX_AXES], start;
  double turns[XDIT_ROTARY_MAX_PAIRS];  // frequency / 2 pi
  uint8_t axis[XDIT_ROTARY_MAX_PAIRS];
};

// Position of token (b, row) along `axis`.
__device__ __forceinline__ double position(const RotaryArgs& a, int b, int row, int axis) {
  if (a.pos_kind == XDIT_POS_GRID) {
    // the last axis runs fastest; tokens behind the grid (padding of a shard) stay at the origin
    int64_t n = a.start + row, below = 1, volume = 1;
    for (int i = 0; i < a.axes; ++i) {
      volume *= a.grid[i];
      if (i > axis) below *= a.grid[i];
    }
    return n < volume ? (double)(n / below % a.grid[axis]) : 0.0;
  }
  const int64_t at = b * a.pos_sb + row * a.pos_srow + axis * a.pos_saxis;
  if (a.pos_kind == XDIT_POS_I32) return (double)__ldg(reinterpret_cast<const int32_t*>(a.pos) + at);
  if (a.pos_kind == XDIT_POS_I64) return (double)__ldg(reinterpret_cast<const long long*>(a.pos) + at);
  return (double)__ldg(reinterpret_cast<const float*>(a.pos) + at);
}

__device__ __forceinline__ void turn(const RotaryArgs& a, int b, int row, int pair, float& c, float& s) {
  const double t = position(a, b, row, a.axis[pair]) * a.turns[pair];
  sincospif((float)(2.0 * (t - rint(t))), &s, &c);
}

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
template <typename T, int V> struct alignas(sizeof(T) * V) Vec { T x[V]; };

// A slot is what one thread owns of a head.  Interleaved pairs: one vector of V elements (V/2 pairs; for
// V = 1 one pair in two scalar accesses).  Halves: the vectors at i and i + rot/2.  Slots behind the
// rotated part hold one vector that is copied.
template <typename T, int V, bool HALVES>
__global__ void __launch_bounds__(kThreads) rotary_axes_kernel(const __grid_constant__ RotaryArgs a) {
  constexpr bool kTwo = HALVES || V == 1;        // two accesses per rotating slot
  constexpr int kPairs = kTwo ? V : V / 2;       // pairs per rotating slot
  using Vt = Vec<T, V>;
  const int64_t item = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int64_t token = item / a.slots;
  if (token >= a.rows * a.splits) return;
  const int slot = (int)(item - token * a.slots);
  const int64_t r = token / a.splits;
  const int split = (int)(token - r * a.splits);
  const int b = (int)(r / a.s), row = (int)(r - (int64_t)b * a.s);
  const int rotating = a.rot / 2 / kPairs;
  const bool rotates = slot < rotating;
  int at0, at1 = 0;
  if (!rotates) at0 = a.rot + (slot - rotating) * V;
  else if (HALVES) { at0 = slot * V; at1 = at0 + a.rot / 2; }
  else if (V == 1) { at0 = 2 * slot; at1 = at0 + 1; }
  else at0 = slot * V;
  float c[kPairs], s[kPairs];
#pragma unroll
  for (int p = 0; p < kPairs; ++p) { c[p] = 1.f; s[p] = 0.f; }
  if (rotates) {
#pragma unroll
    for (int p = 0; p < kPairs; ++p) turn(a, b, row, slot * kPairs + p, c[p], s[p]);
  }
  const int first = split * a.per_split, last = min(first + a.per_split, a.heads[0] + a.heads[1]);
  for (int h0 = first; h0 < last; h0 += kUnroll) {
    Vt x[kUnroll], y[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int g = h0 + u;
      if (g >= last) break;
      const int t = g >= a.heads[0], h = t ? g - a.heads[0] : g;
      const T* src = reinterpret_cast<const T*>(a.src[t]) + b * a.ss_b[t] + h * a.ss_h[t] + row * a.ss_row[t];
      x[u] = *reinterpret_cast<const Vt*>(src + at0);
      if (kTwo && rotates) y[u] = *reinterpret_cast<const Vt*>(src + at1);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int g = h0 + u;
      if (g >= last) break;
      const int t = g >= a.heads[0], h = t ? g - a.heads[0] : g;
      T* dst = reinterpret_cast<T*>(a.dst[t]) + b * a.ds_b[t] + h * a.ds_h[t] + row * a.ds_row[t];
      if (rotates) {
#pragma unroll
        for (int p = 0; p < kPairs; ++p) {
          T& ta = kTwo ? x[u].x[p] : x[u].x[2 * p];
          T& tb = kTwo ? y[u].x[p] : x[u].x[(2 * p + 1) % V];
          const float va = Io<T>::get(ta), vb = Io<T>::get(tb);
          ta = Io<T>::put(va * c[p] - vb * s[p]);
          tb = Io<T>::put(va * s[p] + vb * c[p]);
        }
      }
      *reinterpret_cast<Vt*>(dst + at0) = x[u];
      if (kTwo && rotates) *reinterpret_cast<Vt*>(dst + at1) = y[u];
    }
  }
}

// cos and sin as the attention prologue takes them: fp32 [s, D], each value at both elements of its
// interleaved pair; (1, 0) behind the rotated part.
__global__ void __launch_bounds__(kThreads) rotary_tables_kernel(const __grid_constant__ RotaryArgs a, float* cos,
                                                                 float* sin) {
  const int64_t item = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int64_t row = item / (a.D / 2);
  if (row >= a.s) return;
  const int pair = (int)(item - row * (a.D / 2));
  float c = 1.f, s = 0.f;
  if (2 * pair < a.rot) turn(a, 0, (int)row, pair, c, s);
  *reinterpret_cast<float2*>(cos + row * a.D + 2 * pair) = make_float2(c, c);
  *reinterpret_cast<float2*>(sin + row * a.D + 2 * pair) = make_float2(s, s);
}

int fill_positions(RotaryArgs& a, const xdit_rotary_positions& p, const char* who) {
  if (p.pairs < 1 || p.pairs > XDIT_ROTARY_MAX_PAIRS || p.axes < 1 || p.axes > XDIT_ROTARY_MAX_AXES) {
    set_error("%s: %d pairs (1..%d) on %d axes (1..%d)", who, p.pairs, XDIT_ROTARY_MAX_PAIRS, p.axes, XDIT_ROTARY_MAX_AXES);
    return XDIT_E_SHAPE;
  }
  if (!p.frequencies || !p.axis) { set_error("%s: NULL frequencies or axis", who); return XDIT_E_NULL; }
  if (p.kind < XDIT_POS_GRID || p.kind > XDIT_POS_F32) { set_error("%s: unknown kind of positions %d", who, p.kind); return XDIT_E_DTYPE; }
  for (int i = 0; i < p.pairs; ++i) {
    if (p.axis[i] >= p.axes) { set_error("%s: pair %d is on axis %d of %d", who, i, p.axis[i], p.axes); return XDIT_E_SHAPE; }
    a.turns[i] = p.frequencies[i] / 6.283185307179586476925286766559;
    a.axis[i] = p.axis[i];
  }
  a.rot = 2 * p.pairs;
  a.axes = p.axes;
  a.pos_kind = p.kind;
  if (p.kind == XDIT_POS_GRID) {
    int64_t volume = 1;
    for (int i = 0; i < p.axes; ++i) {
      if (p.grid[i] < 1 || p.grid[i] > (1ll << 40) / volume) { set_error("%s: grid side %lld", who, (long long)p.grid[i]); return XDIT_E_SHAPE; }
      volume *= a.grid[i] = p.grid[i];
    }
    if (p.start < 0 || p.start > (1ll << 40)) { set_error("%s: start %lld", who, (long long)p.start); return XDIT_E_SHAPE; }
    a.start = p.start;
  } else {
    if (!p.positions) { set_error("%s: NULL positions", who); return XDIT_E_NULL; }
    a.pos = p.positions;
    a.pos_sb = p.stride_b;
    a.pos_srow = p.stride_row;
    a.pos_saxis = p.stride_axis;
  }
  return XDIT_OK;
}

template <typename T, int V>
cudaError_t launch(const RotaryArgs& a, bool halves, int64_t blocks, cudaStream_t stream) {
  if (halves) rotary_axes_kernel<T, V, true><<<(unsigned)blocks, kThreads, 0, stream>>>(a);
  else rotary_axes_kernel<T, V, false><<<(unsigned)blocks, kThreads, 0, stream>>>(a);
  return cudaGetLastError();
}

}  // namespace

int launch_rotary(const xdit_rotary_params& p, cudaStream_t stream) {
  RotaryArgs a;
  memset(&a, 0, sizeof(a));
  int rc = fill_positions(a, p.pos, "xdit_rotary_axes");
  if (rc) return rc;
  const int es = dtype_size(p.dtype);
  if (!es) { set_error("xdit_rotary_axes: bad dtype %d", p.dtype); return XDIT_E_DTYPE; }
  if (p.B < 0 || p.s < 0 || p.H < 1 || p.Hk < 0 || p.D < 1 || p.D > 4096 || a.rot > p.D) {
    set_error("xdit_rotary_axes: B=%d s=%d H=%d Hk=%d D=%d, %d elements rotated", p.B, p.s, p.H, p.Hk, p.D, a.rot);
    return XDIT_E_SHAPE;
  }
  if (p.B == 0 || p.s == 0) return XDIT_OK;
  if (!p.q || !p.out_q || (p.Hk && (!p.k || !p.out_k))) { set_error("xdit_rotary_axes: NULL q, k or output"); return XDIT_E_NULL; }
  int sms = 0;
  if ((rc = check_device(&sms))) return rc;
  const int halves = p.halves != 0;
  a.src[0] = (const char*)p.q; a.src[1] = (const char*)p.k;
  a.dst[0] = (char*)p.out_q; a.dst[1] = (char*)p.out_k;
  a.heads[0] = p.H; a.heads[1] = p.Hk;
  a.rows = (int64_t)p.B * p.s;
  a.s = p.s; a.D = p.D;
  // The widest vector that all addresses, strides and the split of a head into pairs allow.
  uint64_t low = 0;  // low bits of everything a vector access starts from, in bytes
  for (int t = 0; t < (p.Hk ? 2 : 1); ++t) {
    a.ss_b[t] = p.stride_b[t]; a.ss_h[t] = p.stride_h[t]; a.ss_row[t] = p.stride_row[t];
    a.ds_b[t] = p.out_stride_b[t]; a.ds_h[t] = p.out_stride_h[t]; a.ds_row[t] = p.out_stride_row[t];
    low |= (uint64_t)(uintptr_t)a.src[t] | (uint64_t)(uintptr_t)a.dst[t];
    if (p.B > 1) low |= (uint64_t)(a.ss_b[t] | a.ds_b[t]) * es;
    if (a.heads[t] > 1) low |= (uint64_t)(a.ss_h[t] | a.ds_h[t]) * es;
    if (p.s > 1) low |= (uint64_t)(a.ss_row[t] | a.ds_row[t]) * es;
  }
  if (low % es) { set_error("xdit_rotary_axes: a pointer is not aligned to its elements"); return XDIT_E_ALIGN; }
  int V = 16 / es;
  const int whole = halves ? a.rot / 2 : a.rot;
  while (V > 1 && ((low % (V * es)) || whole % V || (p.D - a.rot) % V)) V /= 2;
  const int per = (halves || V == 1) ? V : V / 2;  // pairs of a rotating slot
  a.slots = a.rot / 2 / per + (p.D - a.rot) / V;
  // Threads walk all heads unless there are too few tokens to fill the GPU: then the heads are split until
  // about 2048 threads per SM are at work (the angles are then computed once per split).
  const int heads = p.H + p.Hk;
  const int64_t items = a.rows * a.slots;
  int64_t splits = ((int64_t)sms * 2048 + items - 1) / items;
  if (splits > heads) splits = heads;
  a.per_split = (int)((heads + splits - 1) / splits);
  a.splits = (heads + a.per_split - 1) / a.per_split;
  const int64_t blocks = (items * a.splits + kThreads - 1) / kThreads;
  if (blocks > 0x7fffffffll) { set_error("xdit_rotary_axes: too many tokens"); return XDIT_E_SHAPE; }
  cudaError_t e;
#define XDIT_LAUNCH_ROTARY(T)                                          \
  (V == 8 ? launch<T, 8>(a, halves, blocks, stream) : V == 4 ? launch<T, 4>(a, halves, blocks, stream) \
   : V == 2 ? launch<T, 2>(a, halves, blocks, stream) : launch<T, 1>(a, halves, blocks, stream))
  if (p.dtype == XDIT_BF16) e = XDIT_LAUNCH_ROTARY(__nv_bfloat16);
  else if (p.dtype == XDIT_F16) e = XDIT_LAUNCH_ROTARY(__half);
  else e = V == 4 ? launch<float, 4>(a, halves, blocks, stream) : V == 2 ? launch<float, 2>(a, halves, blocks, stream)
                                                              : launch<float, 1>(a, halves, blocks, stream);
#undef XDIT_LAUNCH_ROTARY
  if (e != cudaSuccess) return cuda_fail(e, "rotary_axes_kernel launch");
  return XDIT_OK;
}

int launch_rotary_tables(const xdit_rotary_positions& pos, float* cos, float* sin, int32_t s, int32_t D,
                         cudaStream_t stream) {
  RotaryArgs a;
  memset(&a, 0, sizeof(a));
  int rc = fill_positions(a, pos, "xdit_rotary_tables");
  if (rc) return rc;
  if (s < 0 || D < 2 || D % 2 || D > 4096 || a.rot > D) {
    set_error("xdit_rotary_tables: s=%d D=%d, %d elements rotated", s, D, a.rot);
    return XDIT_E_SHAPE;
  }
  if (s == 0) return XDIT_OK;
  if (!cos || !sin) { set_error("xdit_rotary_tables: NULL cos or sin"); return XDIT_E_NULL; }
  if (((uintptr_t)cos | (uintptr_t)sin) & 7) { set_error("xdit_rotary_tables: cos and sin need 8-byte alignment"); return XDIT_E_ALIGN; }
  if ((rc = check_device(nullptr))) return rc;
  a.s = s; a.D = D;
  const int64_t blocks = ((int64_t)s * (D / 2) + kThreads - 1) / kThreads;
  if (blocks > 0x7fffffffll) { set_error("xdit_rotary_tables: too many tokens"); return XDIT_E_SHAPE; }
  rotary_tables_kernel<<<(unsigned)blocks, kThreads, 0, stream>>>(a, cos, sin);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "rotary_tables_kernel launch");
  return XDIT_OK;
}

}  // namespace xdit

using namespace xdit;

extern "C" {

int xdit_rotary_axes(const struct xdit_rotary_params* p, void* stream) {
  if (!p) { set_error("xdit_rotary_axes: NULL params"); return XDIT_E_NULL; }
  return launch_rotary(*p, (cudaStream_t)stream);
}

int xdit_rotary_tables(const struct xdit_rotary_positions* pos, float* cos, float* sin, int32_t s, int32_t D,
                       void* stream) {
  if (!pos) { set_error("xdit_rotary_tables: NULL positions"); return XDIT_E_NULL; }
  return launch_rotary_tables(*pos, cos, sin, s, D, (cudaStream_t)stream);
}

}  // extern "C"
