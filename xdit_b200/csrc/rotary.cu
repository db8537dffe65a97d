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
// HBM-bound: q and k are read and written once.  A CTA takes a few tokens and many heads of q and k: it computes the
// tokens' angles once, into shared memory, while its first vectors are on their way, and then walks its vectors in
// the order in which they lie in memory (heads of a token, or tokens of a head, whichever are nearer), so that
// loads and stores cover runs of 4 KB.  Tokens share a CTA because 64-bit angles cost more than a head's rotation does:
// with every thread taking its own, q and k of 75,600 tokens x 40 heads of 128 in bf16 (3.10 GB) took 850 us; they take
// 494-506 us (6.1-6.3 TB/s, 0.94-0.96 of a copy), half of the issue slots used.  Four vectors ahead of a thread in 128 registers were
// slower than one ahead in 32 with seven CTAs on an SM.  A token or two are bound by the launch.
#include <cstring>

#include "common.cuh"

namespace xdit {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTokens = 16; // tokens of a CTA

struct RotaryArgs {
  const char* src[2];
  char* dst[2];
  int64_t ss_b[2], ss_h[2], ss_row[2];  // elements
  int64_t ds_b[2], ds_h[2], ds_row[2];
  int32_t heads[2];
  int32_t s, D, rot;
  int32_t slots;       // vectors of a head (pairs of vectors where a rotation takes two)
  int32_t tokens;      // tokens of a CTA, all of one sample
  int32_t blocks_s;    // CTAs along the tokens of a sample
  int32_t per_split;   // heads of a CTA, all of q or all of k
  int32_t splits_q;    // CTAs along the heads of q; those of k follow
  int32_t heads_first; // a token's heads lie nearer to each other than a head's tokens
  // positions
  const void* pos;
  int64_t pos_sb, pos_srow, pos_saxis;
  int32_t pos_kind, axes;
  int64_t grid[XDIT_ROTARY_MAX_AXES], start;
  int32_t grid_small;  // the grid's tokens can be counted in 32 bits
  double turns[XDIT_ROTARY_MAX_PAIRS];  // frequency / 2 pi
  uint8_t axis[XDIT_ROTARY_MAX_PAIRS];
};

template <typename I>
__device__ __forceinline__ double grid_position(const RotaryArgs& a, I n, int axis) {
  // the last axis runs fastest; tokens behind the grid (padding of a shard) stay at the origin
  I below = 1, volume = 1;
  for (int i = 0; i < a.axes; ++i) {
    volume *= (I)a.grid[i];
    if (i > axis) below *= (I)a.grid[i];
  }
  return n < volume ? (double)(n / below % (I)a.grid[axis]) : 0.0;
}
// Position of token (b, row) along `axis`.
__device__ __forceinline__ double position(const RotaryArgs& a, int b, int row, int axis) {
  if (a.pos_kind == XDIT_POS_GRID)
    return a.grid_small ? grid_position<uint32_t>(a, (uint32_t)(a.start + row), axis) : grid_position<uint64_t>(a, (uint64_t)(a.start + row), axis);
  const int64_t at = b * a.pos_sb + row * a.pos_srow + axis * a.pos_saxis;
  if (a.pos_kind == XDIT_POS_I32) return (double)__ldg(reinterpret_cast<const int32_t*>(a.pos) + at);
  if (a.pos_kind == XDIT_POS_I64) return (double)__ldg(reinterpret_cast<const long long*>(a.pos) + at);
  return (double)__ldg(reinterpret_cast<const float*>(a.pos) + at);
}
__device__ __forceinline__ void turn(double position, double turns, float& c, float& s) {
  const double t = position * turns;
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
template <typename T, int V> struct alignas(sizeof(T) * V < 16 ? sizeof(T) * V : 16) Vec { T x[V]; };
// What a slot's access moves: whole words, so that the compiler does not take 16-bit values apart.
template <int BYTES> struct RawOf { using type = Vec<uint32_t, BYTES / 4>; };
template <> struct RawOf<2> { using type = Vec<uint16_t, 1>; };

// Two 16-bit values in a word <-> fp32.
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
__device__ __forceinline__ void rotate(float& x, float& y, float c, float s) {
  const float z = x;
  x = x * c - y * s;
  y = z * s + y * c;
}

// A slot is one thread's part of a head.  Interleaved pairs: one vector of V elements (V/2 pairs; for
// V = 1 one pair in two scalar accesses).  Halves: the vectors at i and i + rot/2.  Slots behind the
// rotated part hold one vector that is copied.  A thread keeps its slot and steps over (token, head) with
// constant strides: what is left per vector is the rotation itself.
template <typename T, int V, bool HALVES>
__global__ void __launch_bounds__(kThreads, HALVES ? 5 : 7) rotary_axes_kernel(const __grid_constant__ RotaryArgs a) {
  extern __shared__ __align__(16) float angles[];  // cos [tokens][pairs], sin [tokens][pairs]
  __shared__ double places[kMaxTokens * XDIT_ROTARY_MAX_AXES], turns[XDIT_ROTARY_MAX_PAIRS];
  __shared__ uint8_t axis[XDIT_ROTARY_MAX_PAIRS];
  constexpr bool kTwo = HALVES || V == 1;   // two accesses per rotating slot
  constexpr int kPairs = kTwo ? V : V / 2;  // pairs per rotating slot
  using Vt = typename RawOf<sizeof(T) * V>::type;
  using Ct = Vec<float, kPairs>;
  const int b = blockIdx.x / a.blocks_s, row0 = (blockIdx.x - b * a.blocks_s) * a.tokens;
  const int t = (int)blockIdx.y >= a.splits_q, head0 = ((int)blockIdx.y - (t ? a.splits_q : 0)) * a.per_split;
  const int tokens = min(a.tokens, a.s - row0), heads = min(a.per_split, a.heads[t] - head0);
  const int pairs = a.rot / 2, rotating = pairs / kPairs;
  float* cosines = angles;
  float* sines = angles + a.tokens * pairs;
  const T* src = reinterpret_cast<const T*>(a.src[t]) + b * a.ss_b[t] + head0 * a.ss_h[t] + row0 * a.ss_row[t];
  T* dst = reinterpret_cast<T*>(a.dst[t]) + b * a.ds_b[t] + head0 * a.ds_h[t] + row0 * a.ds_row[t];
  // (outer, inner) = (token, head) or (head, token), whichever is the order in memory
  const int n_in = a.heads_first ? heads : tokens, n_out = a.heads_first ? tokens : heads;
  // offsets inside a CTA's part fit 32 bits: the launch sees to it
  const int s_in = (int)(a.heads_first ? a.ss_h[t] : a.ss_row[t]), s_out = (int)(a.heads_first ? a.ss_row[t] : a.ss_h[t]);
  const int d_in = (int)(a.heads_first ? a.ds_h[t] : a.ds_row[t]), d_out = (int)(a.heads_first ? a.ds_row[t] : a.ds_h[t]);
  const int width = min(a.slots, kThreads), rows = kThreads / width;  // threads along a head, heads side by side
  const int step_in = rows % n_in, step_out = rows / n_in;
  const int s_step = step_in * s_in + step_out * s_out, s_wrap = s_out - n_in * s_in;
  const int d_step = step_in * d_in + step_out * d_out, d_wrap = d_out - n_in * d_in;
  const int y0 = threadIdx.x / width, total = n_in * n_out;
  bool ready = false;
  for (int slot0 = 0; slot0 < a.slots; slot0 += width) {
    const int slot = slot0 + (int)threadIdx.x - y0 * width;
    const bool rotates = slot < rotating;
    int at0 = slot * V, at1 = 0;
    if (!rotates) at0 = a.rot + (slot - rotating) * V;
    else if (HALVES) at1 = at0 + pairs;
    else if (V == 1) { at0 = 2 * slot; at1 = at0 + 1; }
    const int apart = at1 - at0;
    int in = y0 % n_in, out = y0 / n_in, y = slot < a.slots && y0 < rows ? y0 : total;
    int so = in * s_in + out * s_out + at0, to = in * d_in + out * d_out + at0;
    Vt x, w;
    auto load = [&]() {
      if (y >= total) return;
      x = *reinterpret_cast<const Vt*>(src + so);
      if (kTwo && rotates) w = *reinterpret_cast<const Vt*>(src + so + apart);
    };
    load();
    if (!ready) {  // while the first vectors are on their way
      for (int i = threadIdx.x; i < tokens * a.axes; i += kThreads)
        places[i] = position(a, b, row0 + i / a.axes, i % a.axes);
      for (int i = threadIdx.x; i < pairs; i += kThreads) {  // an argument read at a place of each lane's own is slow
        turns[i] = a.turns[i];
        axis[i] = a.axis[i];
      }
      __syncthreads();
      for (int i = threadIdx.x; i < tokens * pairs; i += kThreads) {
        const int n = i / pairs, pair = i - n * pairs;
        turn(places[n * a.axes + axis[pair]], turns[pair], cosines[i], sines[i]);
      }
      __syncthreads();
      ready = true;
    }
    while (y < total) {
      Vt o = x, o2 = w;
      const int angle = (a.heads_first ? out : in) * pairs + slot * kPairs;
      T* d = dst + to;
      y += rows;
      in += step_in; out += step_out; so += s_step; to += d_step;
      if (in >= n_in) { in -= n_in; ++out; so += s_wrap; to += d_wrap; }
      load();  // the next vector, while this one turns
      if (rotates) {
        const Ct c = *reinterpret_cast<const Ct*>(cosines + angle);
        const Ct s = *reinterpret_cast<const Ct*>(sines + angle);
        if constexpr (sizeof(T) == 2 && V > 1) {
#pragma unroll
          for (int i = 0; i < V / 2; ++i) {
            float x0, x1, y0, y1;
            Word<T>::get(o.x[i], x0, x1);
            if constexpr (HALVES) {
              Word<T>::get(o2.x[i], y0, y1);
              rotate(x0, y0, c.x[2 * i], s.x[2 * i]);
              rotate(x1, y1, c.x[2 * i + 1], s.x[2 * i + 1]);
              o2.x[i] = Word<T>::put(y0, y1);
            } else {
              rotate(x0, x1, c.x[i], s.x[i]);
            }
            o.x[i] = Word<T>::put(x0, x1);
          }
        } else {  // fp32, or one 16-bit value in an access
          T* ta = reinterpret_cast<T*>(&o);
          T* tb = reinterpret_cast<T*>(&o2);
#pragma unroll
          for (int i = 0; i < kPairs; ++i) {
            T& va = kTwo ? ta[i] : ta[2 * i];
            T& vb = kTwo ? tb[i] : ta[(2 * i + 1) % V];
            float x0 = Io<T>::get(va), x1 = Io<T>::get(vb);
            rotate(x0, x1, c.x[i], s.x[i]);
            va = Io<T>::put(x0);
            vb = Io<T>::put(x1);
          }
        }
      }
      *reinterpret_cast<Vt*>(d) = o;
      if (kTwo && rotates) *reinterpret_cast<Vt*>(d + apart) = o2;
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
  if (2 * pair < a.rot) turn(position(a, 0, (int)row, a.axis[pair]), a.turns[pair], c, s);
  *reinterpret_cast<float2*>(cos + row * a.D + 2 * pair) = make_float2(c, c);
  *reinterpret_cast<float2*>(sin + row * a.D + 2 * pair) = make_float2(s, s);
}

// Without `tokens` there may be no positions to point at.
int fill_positions(RotaryArgs& a, const xdit_rotary_positions& p, bool tokens, const char* who) {
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
    a.grid_small = volume < (1ll << 31) && p.start < (1ll << 31);  // start + row stays below 2^32
  } else {
    if (!p.positions && tokens) { set_error("%s: NULL positions", who); return XDIT_E_NULL; }
    a.pos = p.positions;
    a.pos_sb = p.stride_b;
    a.pos_srow = p.stride_row;
    a.pos_saxis = p.stride_axis;
  }
  return XDIT_OK;
}

template <typename T, int V>
cudaError_t launch(const RotaryArgs& a, bool halves, dim3 grid, cudaStream_t stream) {
  const size_t smem = (size_t)a.tokens * a.rot * sizeof(float);
  if (halves) rotary_axes_kernel<T, V, true><<<grid, kThreads, smem, stream>>>(a);
  else rotary_axes_kernel<T, V, false><<<grid, kThreads, smem, stream>>>(a);
  return cudaGetLastError();
}

}  // namespace

int launch_rotary(const xdit_rotary_params& p, cudaStream_t stream) {
  RotaryArgs a;
  memset(&a, 0, sizeof(a));
  int rc = fill_positions(a, p.pos, p.B > 0 && p.s > 0, "xdit_rotary_axes");
  if (rc) return rc;
  const int es = dtype_size(p.dtype);
  if (!es) { set_error("xdit_rotary_axes: bad dtype %d", p.dtype); return XDIT_E_DTYPE; }
  if (p.B < 0 || p.s < 0 || p.H < 1 || p.Hk < 0 || p.D < 1 || p.D > 4096 || a.rot > p.D) {
    set_error("xdit_rotary_axes: B=%d s=%d H=%d Hk=%d D=%d, %d elements rotated", p.B, p.s, p.H, p.Hk, p.D, a.rot);
    return XDIT_E_SHAPE;
  }
  if (p.B == 0 || p.s == 0) return XDIT_OK;
  if (!p.q || !p.out_q || (p.Hk && (!p.k || !p.out_k))) { set_error("xdit_rotary_axes: NULL q, k or output"); return XDIT_E_NULL; }
  const int halves = p.halves != 0;
  a.src[0] = (const char*)p.q; a.src[1] = (const char*)p.k;
  a.dst[0] = (char*)p.out_q; a.dst[1] = (char*)p.out_k;
  a.heads[0] = p.H; a.heads[1] = p.Hk;
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
  for (int t = 0; t < (p.Hk ? 2 : 1); ++t)
    if ((p.B > 1 && !a.ds_b[t]) || (a.heads[t] > 1 && !a.ds_h[t]) || (p.s > 1 && !a.ds_row[t])) {
      set_error("xdit_rotary_axes: an output holds several tokens or heads in one place");
      return XDIT_E_SHAPE;
    }
  if (p.Hk && p.out_q == p.out_k) { set_error("xdit_rotary_axes: q and k have one output"); return XDIT_E_SHAPE; }
  if (p.Hk && (p.out_q == p.k || p.out_k == p.q)) { set_error("xdit_rotary_axes: an output lies on the other input"); return XDIT_E_SHAPE; }
  for (int t = 0; t < (p.Hk ? 2 : 1); ++t)
    if (a.src[t] == a.dst[t] && ((p.B > 1 && a.ss_b[t] != a.ds_b[t]) || (a.heads[t] > 1 && a.ss_h[t] != a.ds_h[t]) ||
                                 (p.s > 1 && a.ss_row[t] != a.ds_row[t]))) {
      set_error("xdit_rotary_axes: an output lies on its input with other strides");
      return XDIT_E_SHAPE;
    }
  if (low % es) { set_error("xdit_rotary_axes: a pointer is not aligned to its elements"); return XDIT_E_ALIGN; }
  int sms = 0;
  if ((rc = check_device(&sms))) return rc;
  int V = 16 / es;
  const int whole = halves ? a.rot / 2 : a.rot;
  while (V > 1 && ((low % (V * es)) || whole % V || (p.D - a.rot) % V)) V /= 2;
  const int per_slot = (halves || V == 1) ? V : V / 2;  // pairs of a rotating slot
  a.slots = a.rot / 2 / per_slot + (p.D - a.rot) / V;
  // A CTA takes 16 tokens and all heads of q or of k; fewer tokens, and then fewer heads, while there are not two CTAs
  // for every SM.
  a.heads_first = p.H > 1 && a.ss_h[0] < a.ss_row[0];
  a.tokens = kMaxTokens;
  auto ctas = [&](int per) {
    return (int64_t)p.B * ((p.s + a.tokens - 1) / a.tokens) * ((p.H + per - 1) / per + (p.Hk + per - 1) / per);
  };
  int per = p.H > p.Hk ? p.H : p.Hk;
  while (a.tokens > 1 && ctas(per) < 2 * sms) a.tokens /= 2;
  while (per > 1 && ctas(per) < 2 * sms && a.tokens * (int64_t)per * a.slots > kThreads) per = (per + 1) / 2;
  // a CTA counts its offsets in 32 bits
  auto reach = [&]() {
    int64_t far = 0;
    for (int t = 0; t < 2; ++t) {
      const int64_t in = a.tokens * a.ss_row[t] + per * a.ss_h[t], out = a.tokens * a.ds_row[t] + per * a.ds_h[t];
      far = in > far ? in : far;
      far = out > far ? out : far;
    }
    return far + p.D;
  };
  while (a.tokens > 1 && reach() > 0x3fffffffll) a.tokens /= 2;
  while (per > 1 && reach() > 0x3fffffffll) per = (per + 1) / 2;
  a.blocks_s = (p.s + a.tokens - 1) / a.tokens;
  a.per_split = per;
  a.splits_q = (p.H + per - 1) / per;
  const int splits = a.splits_q + (p.Hk + per - 1) / per;
  if ((int64_t)p.B * a.blocks_s > 0x7fffffffll || splits > 65535 || (int64_t)a.tokens * per > 0x3fffffffll) {
    set_error("xdit_rotary_axes: too many tokens or heads");
    return XDIT_E_SHAPE;
  }
  const dim3 blocks_grid((unsigned)(p.B * a.blocks_s), splits);
  cudaError_t e;
#define XDIT_LAUNCH_ROTARY(T)                                          \
  (V == 8 ? launch<T, 8>(a, halves, blocks_grid, stream) : V == 4 ? launch<T, 4>(a, halves, blocks_grid, stream) \
   : V == 2 ? launch<T, 2>(a, halves, blocks_grid, stream) : launch<T, 1>(a, halves, blocks_grid, stream))
  if (p.dtype == XDIT_BF16) e = XDIT_LAUNCH_ROTARY(__nv_bfloat16);
  else if (p.dtype == XDIT_F16) e = XDIT_LAUNCH_ROTARY(__half);
  else e = V == 4 ? launch<float, 4>(a, halves, blocks_grid, stream) : V == 2 ? launch<float, 2>(a, halves, blocks_grid, stream)
                                                              : launch<float, 1>(a, halves, blocks_grid, stream);
#undef XDIT_LAUNCH_ROTARY
  if (e != cudaSuccess) return cuda_fail(e, "rotary_axes_kernel launch");
  return XDIT_OK;
}

int launch_rotary_tables(const xdit_rotary_positions& pos, float* cos, float* sin, int32_t s, int32_t D,
                         cudaStream_t stream) {
  RotaryArgs a;
  memset(&a, 0, sizeof(a));
  int rc = fill_positions(a, pos, s > 0, "xdit_rotary_tables");
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
